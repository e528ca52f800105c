// Attention of a sequence's newest rows over its pages (one pass, running maximum
// and sum), instantiated per cache type in attention_{bf16,int8}.hip.
//
// For a row with query q and the tokens j that it sees:
//   s_j = scale q . k_j,  o = sum_j e^(s_j - m) v_j / sum_j e^(s_j - m),  m = max s_j.
// All rows of the query heads that share a key head (up to 16 rows x 64 heads)
// are the columns of 16x16x32 products whose other operand is the cache: S^T = K Q^T
// for a tile of 32 tokens, then O^T += V^T P^T.  The tiles' order (kv_dev.h)
// makes each operand a contiguous 1 KiB load of a wave and leaves the scores of
// 8 consecutive tokens in each lane, which are the k-slots of its P^T operand:
// no value crosses lanes but the maximum of a column (two lane swaps), and
// nothing of a tile goes through LDS.
//
// P is given to the second product as the sum of two bf16 numbers (the rounded
// value and the rounded rest), so that weights keep 16 bits and the result's
// error is that of its own rounding; K, V and Q are exact operands (int8 codes
// are exact in bf16, their scales multiply scores and weights in 32 bits).
//
// A workgroup's waves take the tiles of its part of the length in turn and meet
// in LDS; parts meet through the caller's workspace: each part stores its sums,
// and the one that counts last adds them in part order, so that results do not
// depend on which part that is.
//
// Measured (20 heads over 4 key heads of 128 dims, one row): 600 tokens 6.5 us, 4096 8.4,
// 131072 45.5 (the stream alone 40.2: 6.7 TB/s); 32 sequences of 8192 85 us (6.3 TB/s), int8
// 52; 16 rows of 2 sequences of 4100..8000 18.8 us.  Bound by the cache's stream at long
// contexts (int8 at 5.3 TB/s: 395 VALU instructions a tile to widen codes against 165;
// sequences of uneven lengths by the longest one's parts), by the latency of one load
// chain and of the join at short ones and in 16 rows (where MFMA and softmax issue 6 of
// the 14.4 us).
//
// What a row must not see cannot reach it: masked scores are replaced (not
// added to), places of the last tile past the length are cleared in V.  So a row's
// sum of weights is NaN only where a score that it sees is NaN or +inf, and 0 only
// where all of them are -inf: its result is NaN then, and nothing is read again.  A
// value that is not finite in V would still turn the zero weight of another row of its
// tile into NaN, so other rows whose result is not finite are computed again, one by
// one, over what they see (row_again).
#pragma once

#include "kv_dev.h"

namespace vq {

typedef __bf16 at_bf16x8 __attribute__((ext_vector_type(8)));
typedef float at_f32x4 __attribute__((ext_vector_type(4)));

// Waves of a workgroup that the registers of QT operands of rows leave at most
__host__ __device__ constexpr int at_waves(int D, int qt) { return qt * D <= 256 || (qt == 3 && D == 128) ? 8 : 4; }
// Two workgroups of 8 waves a CU: int8, whose tiles are half as large and take
// half as long again to compute.  A batch then has twice the parts, and what one
// workgroup waits for at its ends another fills (32 sequences of 700 to 16384
// tokens 67.9 us against 75.3; bf16 115.9 against 111.7).
__host__ __device__ constexpr bool at_two(int D, bool i8, int qt) { return i8 && qt * D <= 128; }
// The waves meet in LDS at once, or where that is too small (3 operands of 128
// dims) the upper half goes to the lower half's registers first.
__host__ __device__ constexpr bool at_halves(int D, int qt, int W) { return (size_t)W * qt * 16 * (D + 4) * 4 > 140 * 1024; }
__host__ __device__ constexpr int at_slots(int D, int qt, int W) { return W / (at_halves(D, qt, W) ? 2 : 1); }
constexpr int AT_CNT = 2048;  // counters at the head of the workspace
constexpr int AT_GP = 6;      // parts whose loads a thread has in flight

struct AttnArgs {
    KvArgs c;
    const uint16_t* q;
    uint16_t* out;
    int64_t q_stride, out_stride;
    unsigned* cnt;
    float* part;
    int gqa, qgroups, splits, window, sinks;
    int lrows;      // rows of a group that a workgroup keeps in LDS
    unsigned by_gqa;  // ceil(2^16 / gqa): r / gqa = (r * by_gqa) >> 16 for r < 1024 (gqa <= 64)
    int apart;      // parts are joined by a launch of their own
    float scale;  // times log2 e
};

constexpr int at_qt_max(int D) { return D <= 128 ? 4 : 2; }
// Floats that one part leaves for one group of rows: sums, then {m, l} per row
__host__ __device__ constexpr size_t at_part_floats(int D, int qt) { return (size_t)qt * 16 * (D + 2); }
// LDS: Q's operands; then the waves' sums and {m, l}, or 40 bytes a thread to
// join parts, or 8 a thread and 4 a tile for row_again
inline size_t at_lds_bytes(int D, int qt, int W, int lrows) {
    const size_t S = (size_t)at_slots(D, qt, W), a = S * lrows * (D + 4) * 4 + S * lrows * 8, b = (size_t)W * 64 * 40;
    return (size_t)qt * 16 * D * 2 + (a > b ? a : b);
}

__device__ __forceinline__ float max_over_groups(float v) {
    auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
    r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float sum_over_groups(float v) {
    auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(r[0]) + __uint_as_float(r[1]);
    r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
// 8 int8 codes as an operand of 8 bf16 (exact)
__device__ __forceinline__ at_bf16x8 codes_bf16(uint32_t a, uint32_t b) {
    u32x4 v;
    v.x = f2bf2((float)(int8_t)a, (float)(int8_t)(a >> 8));
    v.y = f2bf2((float)(int8_t)(a >> 16), (float)(int8_t)(a >> 24));
    v.z = f2bf2((float)(int8_t)b, (float)(int8_t)(b >> 8));
    v.w = f2bf2((float)(int8_t)(b >> 16), (float)(int8_t)(b >> 24));
    return __builtin_bit_cast(at_bf16x8, v);
}

// exp2 of a difference to a maximum that is -inf where nothing was seen
__device__ __forceinline__ float part_weight(float m, float M) {
    return m == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f(m - M);
}

// What the row at position p sees
struct Sight {
    int window, sinks;
    __device__ __forceinline__ bool sees(int j, int p) const {
        return j <= p && (window == 0 || j > p - window || j < sinks);
    }
};

// 8 values of 16 or 8 bytes
__device__ __forceinline__ void again_bf16(const u32x4& v, float* f) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = bf16f((w[i >> 1] >> (16 * (i & 1))) & 0xffffu);
}
__device__ __forceinline__ void again_codes(const u32x2& v, float* f) {
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = (float)(int8_t)((i < 4 ? v.x : v.y) >> (8 * (i & 3)));
}

// One row computed on its own over the tokens that it sees, from the maximum m and the sum
// of weights l that the first pass found: weights by the thread of a token, sums by the
// thread of a dim and 8 tokens.  Reached only by rows whose sums are not finite though
// their weights are numbers: values in V that are not, seen or in a seen token's tile, finite
// ones whose sum leaves 32 bits (10^38; their mean does not), and missing pages (which are
// looked for first).  One workgroup reads the row's K and V at the latency of its loads, rows
// side by side where the parts are joined by a launch of their own (65536 tokens of 128 dims
// 3.6 ms), else one after the other (5 rows of 8192 tokens 0.8 ms).
template <int D, bool I8, int NT>
__device__ __forceinline__ void row_again(const AttnArgs& a, int b, int head, const uint16_t* q, uint16_t* o,
                                                    int p, float2 ml, float* lds) {
    constexpr int TILES = NT / KV_TILE, G = NT / D;  // tiles of a chunk of tokens; groups of threads over its octets
    const int tid = (int)threadIdx.x;
    const Sight sight{a.window, a.sinks};
    const int64_t cap = ((int64_t)a.c.width << a.c.tpl) * KV_TILE;
    float* w = lds;                // [NT] weights of a chunk of tokens, -1: not seen
    float* acc = w + NT;           // [NT]
    int* pages = (int*)(acc + NT);  // [TILES]
    // chunks between the first tokens and the window are skipped
    auto between = [&](int64_t j0, int n) { return a.window != 0 && j0 >= a.sinks && j0 + n - 1 <= (int64_t)p - a.window; };
    bool bad = p >= cap;
    if (!bad) {
        for (int64_t tile = tid; tile * KV_TILE <= p; tile += NT)
            if (!between(tile * KV_TILE, KV_TILE) && kv_page(a.c, b, (int)tile) < 0) bad = true;
    }
    bad = __syncthreads_or(bad);
    // (weights of the mean: a sum of them times finite values stays finite)
    const float il = 1.0f / ml.y;
    float sum = 0.0f;
    for (int64_t j0 = 0; j0 <= p && !bad; j0 += NT) {
        if (between(j0, NT)) continue;
        const bool in = j0 + tid <= p && sight.sees((int)(j0 + tid), p);
        float e = -1.0f;
        if (in) {
            const int j = (int)j0 + tid, tile = j / KV_TILE, t = j % KV_TILE;
            const size_t at = kv_tile_at(a.c, kv_page(a.c, b, tile), head, tile), base = at * (KV_TILE * D);
            float s = 0.0f;
#pragma unroll 2
            for (int c = 0; c < D / 8; ++c) {
                float k[8], x[8];
                if constexpr (I8) again_codes(*(const u32x2*)((const int8_t*)a.c.k + base + k_place<true>(t, c)), k);
                else again_bf16(*(const u32x4*)((const uint16_t*)a.c.k + base + k_place<false>(t, c)), k);
                again_bf16(*(const u32x4*)(q + 8 * c), x);
#pragma unroll
                for (int i = 0; i < 8; ++i) s = __builtin_fmaf(x[i], k[i], s);
            }
            if (I8) s *= a.c.ks[at * KV_TILE + t];
            e = __builtin_amdgcn_exp2f(s * a.scale - ml.x) * il;
        }
        __syncthreads();
        w[tid] = e;
        if (tid < TILES) pages[tid] = kv_page(a.c, b, (int)min(j0 / KV_TILE + tid, (int64_t)p / KV_TILE));
        __syncthreads();
        const int d = tid % D;
#pragma unroll 2
        for (int i = tid / D; i < NT / 8; i += G) {
            const int pg = pages[i / 4];  // (4 octets of tokens a tile)
            if (pg < 0) continue;         // (none of its tokens is seen)
            const size_t at = kv_tile_at(a.c, pg, head, (int)(j0 / KV_TILE) + i / 4), base = at * (KV_TILE * D);
            float v[8];
            if constexpr (I8) {
                again_codes(*(const u32x2*)((const int8_t*)a.c.v + base + v_place<true>(8 * (i & 3), d)), v);
#pragma unroll
                for (int x = 0; x < 8; ++x) v[x] *= a.c.vs[at * KV_TILE + 8 * (i & 3) + x];
            } else {
                again_bf16(*(const u32x4*)((const uint16_t*)a.c.v + base + v_place<false>(8 * (i & 3), d)), v);
            }
#pragma unroll
            for (int x = 0; x < 8; ++x) sum = w[8 * i + x] == -1.0f ? sum : __builtin_fmaf(w[8 * i + x], v[x], sum);
        }
    }
    acc[tid] = sum;
    __syncthreads();
    if (tid < D) {
        float v = __uint_as_float(0x7fc00000u);
        if (!bad) {
            v = 0.0f;
            for (int i = tid; i < NT; i += D) v += acc[i];
        }
        o[tid] = f2bf(v);
    }
    __syncthreads();
}

// What a group of rows of a sequence has to look at
struct AttnSeq {
    KvSeq sq;
    int rows;        // of the group
    int len, pos0;   // length, position of the sequence's first row
    int nsink, lo_t, tiles;
    int parts;       // that have tiles
    bool over;       // longer than its table
    __device__ __forceinline__ int tile_of(int v) const { return v < nsink ? v : v - nsink + lo_t; }
};
template <int ROWS, int W>
__device__ __forceinline__ AttnSeq attn_seq(const AttnArgs& a, const KvSeq& sq, int qg) {
    AttnSeq s;
    s.sq = sq;
    s.rows = min(ROWS, sq.n * a.gqa - qg * ROWS);
    const int cap = (a.c.width << a.c.tpl) * KV_TILE;
    s.len = max(0, sq.len);
    s.over = s.len > cap;
    s.pos0 = s.len - sq.n;
    // the tiles that some row sees: those of the first tokens, then the window's
    s.lo_t = s.nsink = 0;
    if (a.window != 0) {
        const int from = max(0, s.pos0 + 1 > a.window ? s.pos0 + 1 - a.window : 0);
        // (a length past the table has no more tiles than it)
        s.nsink = (min(min(a.sinks, from), cap) + KV_TILE - 1) / KV_TILE;
        s.lo_t = max(from / KV_TILE, s.nsink);
    }
    s.tiles = s.nsink + max(0, (min(s.len, cap) + KV_TILE - 1) / KV_TILE - s.lo_t);
    s.parts = max(1, min(a.splits, (s.tiles + W - 1) / W));
    return s;
}

// Row rr of group qg as a result; false where it has to be computed again: its weights are
// numbers, the sums of its values are not finite (0 * x is NaN then)
template <int D, int ROWS>
__device__ __forceinline__ bool attn_store(const AttnArgs& a, const AttnSeq& s, int qg, int head, int rr, int d, at_f32x4 o,
                                           float l) {
    const int r = qg * ROWS + rr, i = (int)((unsigned)r * a.by_gqa >> 16), hh = r - i * a.gqa;
    o = o * (1.0f / l);  // (NaN where l is 0 or NaN)
    bool fine = !(l > 0.0f);
    if (s.pos0 + i < 0) o = at_f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    fine |= o[0] * 0.0f + o[1] * 0.0f + o[2] * 0.0f + o[3] * 0.0f == 0.0f;
    *(u32x2*)(a.out + (size_t)(s.sq.row0 + i) * a.out_stride + (size_t)(head * a.gqa + hh) * D + d) =
        u32x2{f2bf2(o[0], o[1]), f2bf2(o[2], o[3])};
    return fine;
}
template <int D, bool I8, int NT, int ROWS>
__device__ __forceinline__ void attn_again(const AttnArgs& a, const AttnSeq& s, int b, int qg, int head, int rr, float2 ml,
                                           float* lds) {
    const int r = qg * ROWS + rr, i = (int)((unsigned)r * a.by_gqa >> 16), hh = r - i * a.gqa;
    const size_t row = (size_t)s.sq.row0 + i, h = (size_t)(head * a.gqa + hh) * D;
    row_again<D, I8, NT>(a, b, head, a.q + row * a.q_stride + h, a.out + row * a.out_stride + h, s.pos0 + i, ml, lds);
}

// Sums of 8 values (row rr, dims d ..) over parts first, first + step, ...
// Parts are written through to where every XCD sees them (each has an L2 of its
// own) and read back past it, so that no cache is written back or dropped as a
// whole.  Such a load takes over a microsecond: AT_GP parts are in flight together.
struct AttnSum {
    at_f32x4 o0, o1;
    float M, l;
};
template <int D, int ROWS>
__device__ __forceinline__ AttnSum attn_join(__amdgpu_buffer_rsrc_t recs, int rr, int d, int first, int step, int parts) {
    constexpr int PF = (int)at_part_floats(D, ROWS / 16);
    AttnSum s{{0.0f, 0.0f, 0.0f, 0.0f}, {0.0f, 0.0f, 0.0f, 0.0f}, -__builtin_inff(), 0.0f};
    for (int s0 = first; s0 < parts; s0 += AT_GP * step) {
        u32x4 va[AT_GP], vb[AT_GP];
        u32x2 ml[AT_GP];
#pragma unroll
        for (int k = 0; k < AT_GP; ++k) {  // (past the parts: zeros)
            const int p = s0 + k * step, at = p * PF * 4;
            ml[k] = bload8<AUX_SC1>(recs, p < parts ? at + (ROWS * D + 2 * rr) * 4 : OOB);
            va[k] = bload16<AUX_SC1>(recs, p < parts ? at + (rr * D + d) * 4 : OOB);
            vb[k] = bload16<AUX_SC1>(recs, p < parts ? at + (rr * D + d) * 4 + 16 : OOB);
        }
        issue_fence();
        float M = s.M;
#pragma unroll
        for (int k = 0; k < AT_GP; ++k) M = fmaxf(M, s0 + k * step < parts ? __uint_as_float(ml[k].x) : -__builtin_inff());
        const float f0 = part_weight(s.M, M);
        s.o0 *= f0;
        s.o1 *= f0;
        s.l = s.l == s.l ? s.l * f0 : s.l;
        s.M = M;
#pragma unroll
        for (int k = 0; k < AT_GP; ++k) {
            const float f = s0 + k * step < parts ? part_weight(__uint_as_float(ml[k].x), M) : 0.0f, l = __uint_as_float(ml[k].y);
            s.o0 += __builtin_bit_cast(at_f32x4, va[k]) * f;
            s.o1 += __builtin_bit_cast(at_f32x4, vb[k]) * f;
            s.l += l == l ? l * f : l;
        }
    }
    return s;
}
// The groups of threads meet: thread t < 2 * units stores 4 values of unit t % units
// and leaves the row's maximum and sum in ml
template <int D, int ROWS>
__device__ __forceinline__ bool attn_meet(const AttnArgs& a, const AttnSeq& s, int qg, int head, int rr0, float* lds, int NT,
                                          int units, int G, float2& ml) {
    const at_f32x4* jo = (const at_f32x4*)lds;
    const float* jm = lds + 8 * NT;
    const int tid = (int)threadIdx.x, half = tid >= units, u = tid - half * units;
    float M = -__builtin_inff(), l = 0.0f;
    at_f32x4 o = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int k = 0; k < G; ++k) M = fmaxf(M, jm[2 * (k * units + u)]);
    for (int k = 0; k < G; ++k) {
        const float f = part_weight(jm[2 * (k * units + u)], M), lw = jm[2 * (k * units + u) + 1];
        o += jo[half * NT + k * units + u] * f;
        l += lw == lw ? lw * f : lw;
    }
    ml = make_float2(M, l);
    return attn_store<D, ROWS>(a, s, qg, head, rr0 + u / (D / 8), u % (D / 8) * 8 + 4 * half, o, l);
}
__device__ __forceinline__ void attn_lay(float* lds, int NT, const AttnSum& s) {
    at_f32x4* jo = (at_f32x4*)lds;  // [2][NT]
    float* jm = lds + 8 * NT;       // [NT][2]
    jo[threadIdx.x] = s.o0;
    jo[NT + threadIdx.x] = s.o1;
    jm[2 * threadIdx.x] = s.M;
    jm[2 * threadIdx.x + 1] = s.l;
}

template <int D, bool I8, int QT, int W>
__global__ void __launch_bounds__(W * 64) __attribute__((amdgpu_waves_per_eu(at_two(D, I8, QT) ? 4 : 1)))
attn_kernel(AttnArgs a) {
    constexpr int NT = W * 64;
    constexpr int NKB = D / 32, NDB = D / 16, ROWS = QT * 16, ST = D + 4;
    constexpr int NK = I8 ? NKB : 2 * NKB, NV = I8 ? NDB / 2 : NDB;  // 16-byte loads of a lane per tile
    constexpr int SLOTS = at_slots(D, QT, W);
    extern __shared__ __align__(16) u32x4 lq[];  // Q's operands [QT][NKB][64]
    const int LR = a.lrows;
    float* lds = (float*)(lq + QT * NKB * 64);
    float* lo = lds;                    // [SLOTS][LR][ST]
    float* lml = lds + SLOTS * LR * ST;  // [SLOTS][LR][2]
    __shared__ int last_part;
    __shared__ unsigned again[(ROWS + 31) / 32];
    __shared__ float2 again_ml[ROWS];

    const int tid = (int)threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int l16 = lane & 15, g = lane >> 4;
    const int split = (int)blockIdx.x, b = (int)blockIdx.z;
    int head = (int)blockIdx.y, qg = 0;
    if (a.qgroups > 1) {
        qg = head / a.c.kvh;
        head -= qg * a.c.kvh;
    }
    // Part p of P takes tiles (p + k P) W + wave, so that its first tile does not
    // depend on the length (but with a window): its page and the sequence's length
    // are asked for together.
    const int v0 = split * W + wave, stride = a.splits * W;
    int page0 = kv_sload(a.c.table, (size_t)b * a.c.width + min(v0 >> a.c.tpl, a.c.width - 1));
    KvSeq sq = kv_seq(a.c, b);
    asm volatile("" : "+s"(page0), "+s"(sq.len));
    const AttnSeq s = attn_seq<ROWS, W>(a, sq, qg);
    const int rows = s.rows, len = s.len, pos0 = s.pos0, tiles = s.tiles, parts = s.parts;
    if (rows <= 0 || split >= parts) return;

    // Q as the operand with rows as its columns, shared by the waves in LDS
    constexpr int QC = QT * NKB * 64, QN = (QC + NT - 1) / NT;  // 16-byte chunks, of a thread
    u32x4 qv[QN];
#pragma unroll
    for (int k = 0; k < QN; ++k) {
        const int x = tid + k * NT, kb = (x >> 6) % NKB, rr = (x >> 6) / NKB * 16 + (x & 15), r = qg * ROWS + rr;
        const int i = (int)((unsigned)r * a.by_gqa >> 16), hh = r - i * a.gqa;
        qv[k] = u32x4{0u, 0u, 0u, 0u};
        if (rr < rows)
            qv[k] = *(const u32x4*)(a.q + (size_t)(sq.row0 + i) * a.q_stride + (size_t)(head * a.gqa + hh) * D + kb * 32 +
                                    8 * ((x >> 4) & 3));
    }
    int pos[QT];  // position of the lane's row, -1: no row
#pragma unroll
    for (int qt = 0; qt < QT; ++qt) {
        const int rr = qt * 16 + l16;
        pos[qt] = rr < rows ? pos0 + (int)((unsigned)(qg * ROWS + rr) * a.by_gqa >> 16) : -1;
    }

    at_f32x4 O[QT][NDB];
    float m[QT], l[QT];
#pragma unroll
    for (int qt = 0; qt < QT; ++qt) {
        m[qt] = -__builtin_inff();
        l[qt] = 0.0f;
#pragma unroll
        for (int db = 0; db < NDB; ++db) O[qt][db] = at_f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    }
    bool missing = s.over;

    u32x4 kr[NK], vr[NV];
    u32x4 ksc[2], vsc[2];
    constexpr int TB = KV_TILE * D * (I8 ? 1 : 2);  // bytes of a tile
    // A tile that one workgroup reads is not kept (131072 tokens, one row: 58 us
    // instead of 68); several groups of rows read it again from L2.
    constexpr int AUX = QT < at_qt_max(D) && QT <= 2 ? AUX_NT : 0;
    auto load_tile = [&](const void* pool, size_t at, u32x4* r, auto n) {
        const auto t = buf((const uint8_t*)pool + at * TB, TB);
#pragma unroll
        for (int i = 0; i < n(); ++i) {
            const i32x4 w = __builtin_amdgcn_raw_buffer_load_b128(t, lane * 16 + (i & 3) * 1024, (i >> 2) * 4096, AUX);
            r[i] = u32x4{(uint32_t)w.x, (uint32_t)w.y, (uint32_t)w.z, (uint32_t)w.w};
        }
    };
    auto load_scales = [&](const float* pool, size_t at, u32x4* r) {
        const auto t = buf(pool + at * KV_TILE, KV_TILE * 4);
        r[0] = bload16(t, g * 32);
        r[1] = bload16(t, g * 32 + 16);
    };
    auto load_k = [&](int page, int tile) {
        const size_t at = kv_tile_at(a.c, page, head, tile);
        load_tile(a.c.k, at, kr, [] { return NK; });
        if constexpr (I8) load_scales(a.c.ks, at, ksc);
    };
    auto load_v = [&](int page, int tile) {
        const size_t at = kv_tile_at(a.c, page, head, tile);
        load_tile(a.c.v, at, vr, [] { return NV; });
        if constexpr (I8) load_scales(a.c.vs, at, vsc);
    };

    // A tile's K is asked for once the products that read the one before are
    // issued, its V likewise, its page two tiles ahead.  A tile whose page is missing
    // reads page 0 and makes the sums of every row of the wave NaN (row_again sorts them out).
    auto page_of = [&](int v) {
        const int p = v < tiles ? kv_page_uniform(a.c, b, s.tile_of(v)) : 0;
        if (p < 0) missing = true;
        return max(p, 0);
    };
    if (v0 < tiles) {
        int p = page0;
        if (a.window != 0) p = kv_page_uniform(a.c, b, s.tile_of(v0));
        if ((unsigned)p >= (unsigned)a.c.pages) {
            missing = true;
            p = 0;
        }
        load_k(p, s.tile_of(v0));
        load_v(p, s.tile_of(v0));
    }
    int pn, pnn = page_of(v0 + stride);
#pragma unroll
    for (int k = 0; k < QN; ++k)
        if (QC % NT == 0 || tid + k * NT < QC) lq[tid + k * NT] = qv[k];
    lds_barrier();
    for (int v = v0; v < tiles; v += stride) {
        const int tile = s.tile_of(v), next = s.tile_of(v + stride);
        const bool more = v + stride < tiles;
        pn = pnn;
        pnn = page_of(v + 2 * stride);
        issue_fence();  // (Q is read again for each tile: its registers go to K and V)
        if constexpr (I8) {  // (codes are not widened before their tile's turn)
#pragma unroll
            for (int i = 0; i < NK; ++i) asm volatile("" : "+v"(kr[i]));
        }
        at_f32x4 S[QT][2];
#pragma unroll
        for (int qt = 0; qt < QT; ++qt) S[qt][0] = S[qt][1] = at_f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int kb = 0; kb < NKB; ++kb) {
            at_bf16x8 qf[QT];
#pragma unroll
            for (int qt = 0; qt < QT; ++qt) qf[qt] = __builtin_bit_cast(at_bf16x8, lq[(qt * NKB + kb) * 64 + lane]);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                at_bf16x8 k;
                if constexpr (I8) {
                    const u32x4 w = kr[(kb >> 1) * 2 + h];
                    k = kb & 1 ? codes_bf16(w.z, w.w) : codes_bf16(w.x, w.y);
                } else {
                    k = __builtin_bit_cast(at_bf16x8, kr[kb * 2 + h]);
                }
#pragma unroll
                for (int qt = 0; qt < QT; ++qt)
                    S[qt][h] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k, qf[qt], S[qt][h], 0, 0, 0);
            }
        }
        float kscale[8], vscale[8];
        if constexpr (I8) {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                kscale[e] = __uint_as_float(ksc[e >> 2][e & 3]) * a.scale;
                vscale[e] = __uint_as_float(vsc[e >> 2][e & 3]);
            }
        }
        if (more) load_k(pn, next);
        // scores, by token of the lane's eight; tiles that some row does not see whole are masked
        const int j0 = tile * KV_TILE, jl = j0 + 8 * g;
        const bool whole = j0 + KV_TILE - 1 <= pos0 &&
                           (a.window == 0 || j0 > len - 1 - a.window || j0 + KV_TILE <= a.sinks);
        at_bf16x8 ph[QT], pl[QT];
#pragma unroll
        for (int qt = 0; qt < QT; ++qt) {
            float x[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                x[e] = S[qt][e >> 2][e & 3] * (I8 ? kscale[e] : a.scale);
            }
            uint32_t seen = 0xffu;
            if (!whole) {
                const Sight sight{a.window, a.sinks};
                seen = 0;
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const bool in = sight.sees(jl + e, pos[qt]);
                    seen |= in ? 1u << e : 0u;
                    x[e] = in ? x[e] : -__builtin_inff();
                }
            }
            float mt = fmaxf(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])), fmaxf(fmaxf(x[4], x[5]), fmaxf(x[6], x[7])));
            mt = fmaxf(m[qt], max_over_groups(mt));
            const float ms = mt == -__builtin_inff() ? 0.0f : mt;
            const float f = __builtin_amdgcn_exp2f(m[qt] - ms);
            m[qt] = mt;
            float sum = 0.0f;
            float p[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                p[e] = __builtin_amdgcn_exp2f(x[e] - ms);
                sum += p[e];
                if constexpr (I8) p[e] = (seen >> e) & 1 ? p[e] * vscale[e] : 0.0f;
            }
            l[qt] = l[qt] * f + sum;
#pragma unroll
            for (int db = 0; db < NDB; ++db) O[qt][db] *= f;
            u32x4 h, r;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const uint32_t w = f2bf2(p[2 * e], p[2 * e + 1]);
                h[e] = w;
                r[e] = f2bf2(p[2 * e] - bf16f(w & 0xffffu), p[2 * e + 1] - bf16f(w >> 16));
            }
            ph[qt] = __builtin_bit_cast(at_bf16x8, h);
            pl[qt] = __builtin_bit_cast(at_bf16x8, r);
        }
        if (!I8 && j0 + KV_TILE > len) {  // places past the length hold anything
#pragma unroll
            for (int i = 0; i < NV; ++i) {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    vr[i][e] &= (jl + 2 * e < len ? 0xffffu : 0u) | (jl + 2 * e + 1 < len ? 0xffff0000u : 0u);
            }
        }
        if constexpr (I8) {
#pragma unroll
            for (int i = 0; i < NV; ++i) asm volatile("" : "+v"(vr[i]));
        }
#pragma unroll
        for (int db = 0; db < NDB; ++db) {
            at_bf16x8 vv;
            if constexpr (I8) {
                const u32x4 w = vr[db >> 1];
                vv = db & 1 ? codes_bf16(w.z, w.w) : codes_bf16(w.x, w.y);
            } else {
                vv = __builtin_bit_cast(at_bf16x8, vr[db]);
            }
#pragma unroll
            for (int qt = 0; qt < QT; ++qt) {
                O[qt][db] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vv, ph[qt], O[qt][db], 0, 0, 0);
                O[qt][db] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vv, pl[qt], O[qt][db], 0, 0, 0);
            }
        }
        if (more) load_v(pn, next);
    }

    // the waves meet
#pragma unroll
    for (int qt = 0; qt < QT; ++qt) {
        l[qt] = sum_over_groups(l[qt]);
        if (missing) {
#pragma unroll
            for (int db = 0; db < NDB; ++db) O[qt][db][0] = __uint_as_float(0x7fc00000u);
        }
    }
    auto put = [&](int slot) {
#pragma unroll
        for (int qt = 0; qt < QT; ++qt) {
            const int row = slot * LR + qt * 16 + l16;
            if (qt * 16 + l16 >= LR) continue;
            if (g == 0) *(float2*)(lml + 2 * row) = make_float2(m[qt], l[qt]);
#pragma unroll
            for (int db = 0; db < NDB; ++db) *(at_f32x4*)(lo + row * ST + 16 * db + 4 * g) = O[qt][db];
        }
    };
    if constexpr (at_halves(D, QT, W)) {
        if (wave >= SLOTS) put(wave - SLOTS);
        lds_barrier();
        if (wave < SLOTS) {
#pragma unroll
            for (int qt = 0; qt < QT; ++qt) {
                const int row = wave * LR + qt * 16 + l16;
                if (qt * 16 + l16 >= LR) continue;
                const float2 ml = *(const float2*)(lml + 2 * row);
                const float M = fmaxf(m[qt], ml.x), f0 = part_weight(m[qt], M), f1 = part_weight(ml.x, M);
                l[qt] = (l[qt] == l[qt] ? l[qt] * f0 : l[qt]) + (ml.y == ml.y ? ml.y * f1 : ml.y);
                m[qt] = M;
#pragma unroll
                for (int db = 0; db < NDB; ++db)
                    O[qt][db] = O[qt][db] * f0 + *(const at_f32x4*)(lo + row * ST + 16 * db + 4 * g) * f1;
            }
        }
        lds_barrier();
        if (wave < SLOTS) put(wave);
    } else {
        put(wave);
    }
    if (tid < (ROWS + 31) / 32) again[tid] = 0u;
    __syncthreads();

    const int rec = (qg * a.c.batch + b) * a.c.kvh + head;
    constexpr int PF = (int)at_part_floats(D, QT);
    auto once_more = [&](int rr, float2 ml) {  // (threads of one row have the same ml)
        again_ml[rr] = ml;
        atomicOr(&again[rr >> 5], 1u << (rr & 31));
    };
    auto store = [&](int rr, int d, at_f32x4 o, float M, float lt) {
        if (!attn_store<D, ROWS>(a, s, qg, head, rr, d, o, lt)) once_more(rr, make_float2(M, lt));
    };
    const auto recs = buf(a.part + (size_t)rec * a.splits * PF, (uint32_t)(parts * PF * 4));
    for (int i = tid; i < rows * (D / 4); i += NT) {
        const int rr = i / (D / 4), d = i % (D / 4) * 4;
        float M = lml[2 * rr];
#pragma unroll
        for (int w = 1; w < SLOTS; ++w) M = fmaxf(M, lml[2 * (w * LR + rr)]);
        at_f32x4 o = {0.0f, 0.0f, 0.0f, 0.0f};
        float lt = 0.0f;
#pragma unroll
        for (int w = 0; w < SLOTS; ++w) {
            const float f = part_weight(lml[2 * (w * LR + rr)], M), lw = lml[2 * (w * LR + rr) + 1];
            o += *(const at_f32x4*)(lo + (w * LR + rr) * ST + d) * f;
            lt += lw == lw ? lw * f : lw;
        }
        if (parts == 1) {
            store(rr, d, o, M, lt);
        } else {
            bstore16<AUX_SC1>(recs, (split * PF + rr * D + d) * 4, __builtin_bit_cast(u32x4, o));
            if (d == 0)
                bstore8<AUX_SC1>(recs, (split * PF + ROWS * D + 2 * rr) * 4, u32x2{__float_as_uint(M), __float_as_uint(lt)});
        }
    }
    if (parts > 1) {
        if (a.apart) return;
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
        if (tid == 0) {
            const unsigned old = __hip_atomic_fetch_add(a.cnt + rec, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            last_part = old == (unsigned)(parts - 1);
            if (last_part) __hip_atomic_store(a.cnt + rec, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        }
        __syncthreads();
        if (!last_part) return;
        // each group of threads takes every G-th part of all rows, 8 values a thread
        const int units = rows * (D / 8), G = max(1, min(NT / units, (parts + AT_GP - 1) / AT_GP)), grp = G > 1 ? tid / units : 0;
        for (int i = G > 1 ? tid - grp * units : tid; i < units && grp < G; i += NT) {
            const int rr = i / (D / 8), d = i % (D / 8) * 8;
            const AttnSum t = attn_join<D, ROWS>(recs, rr, d, grp, G, parts);
            if (G == 1) {
                store(rr, d, t.o0, t.M, t.l);
                store(rr, d + 4, t.o1, t.M, t.l);
            } else {
                attn_lay(lds, NT, t);
            }
        }
        if (G > 1) {
            __syncthreads();
            float2 ml;
            if (tid < 2 * units && !attn_meet<D, ROWS>(a, s, qg, head, 0, lds, NT, units, G, ml))
                once_more((tid >= units ? tid - units : tid) / (D / 8), ml);
        }
    }
    __syncthreads();
    for (int rr = 0; rr < rows; ++rr)
        if ((again[rr >> 5] >> (rr & 31)) & 1u) attn_again<D, I8, NT, ROWS>(a, s, b, qg, head, rr, again_ml[rr], lds);
}

// The join as a launch of its own: a workgroup per row and group of rows, its
// threads D / 8 values wide and G parts deep.
constexpr int AT_JNT = 256;
template <int D, bool I8, int QT, int W>
__global__ void __launch_bounds__(AT_JNT)
attn_join_kernel(AttnArgs a) {
    constexpr int ROWS = QT * 16, U = D / 8, G = AT_JNT / U;
    __shared__ __align__(16) float lds[AT_JNT * 10];
    __shared__ int again;
    __shared__ float2 again_ml;
    const int b = (int)blockIdx.z, rr = (int)blockIdx.x, tid = (int)threadIdx.x;
    int head = (int)blockIdx.y, qg = 0;
    if (a.qgroups > 1) {
        qg = head / a.c.kvh;
        head -= qg * a.c.kvh;
    }
    const AttnSeq s = attn_seq<ROWS, W>(a, kv_seq(a.c, b), qg);
    if (rr >= s.rows || s.parts == 1) return;
    const int rec = (qg * a.c.batch + b) * a.c.kvh + head;
    constexpr int PF = (int)at_part_floats(D, QT);
    const auto recs = buf(a.part + (size_t)rec * a.splits * PF, (uint32_t)(s.parts * PF * 4));
    attn_lay(lds, AT_JNT, attn_join<D, ROWS>(recs, rr, tid % U * 8, tid / U, G, s.parts));
    if (tid == 0) again = 0;
    __syncthreads();
    float2 ml;
    if (tid < 2 * U && !attn_meet<D, ROWS>(a, s, qg, head, rr, lds, AT_JNT, U, G, ml)) {
        again_ml = ml;
        again = 1;
    }
    __syncthreads();
    if (again) attn_again<D, I8, AT_JNT, ROWS>(a, s, b, qg, head, rr, again_ml, lds);
}

struct AttnFn {
    const void* attn;
    const void* join;
};
template <int D, bool I8, int QT, int W>
inline AttnFn attn_pair() {
    return AttnFn{(const void*)attn_kernel<D, I8, QT, W>, (const void*)attn_join_kernel<D, I8, QT, W>};
}
template <int D, bool I8, int QT>
inline AttnFn attn_of(int W) {
    if constexpr (at_waves(D, QT) == 8)
        if (W == 8) return attn_pair<D, I8, QT, 8>();
    return attn_pair<D, I8, QT, 4>();
}
template <bool I8>
inline AttnFn attn_fn(int D, int qt, int W) {
    switch (D * 8 + qt) {
        case 64 * 8 + 1: return attn_of<64, I8, 1>(W);
        case 64 * 8 + 2: return attn_of<64, I8, 2>(W);
        case 64 * 8 + 3: return attn_of<64, I8, 3>(W);
        case 64 * 8 + 4: return attn_of<64, I8, 4>(W);
        case 128 * 8 + 1: return attn_of<128, I8, 1>(W);
        case 128 * 8 + 2: return attn_of<128, I8, 2>(W);
        case 128 * 8 + 3: return attn_of<128, I8, 3>(W);
        case 128 * 8 + 4: return attn_of<128, I8, 4>(W);
        case 256 * 8 + 1: return attn_of<256, I8, 1>(W);
        case 256 * 8 + 2: return attn_of<256, I8, 2>(W);
        default: return AttnFn{nullptr, nullptr};
    }
}

}  // namespace vq
