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
// A workgroup's 4 waves take every fourth tile of its part of the length and meet
// in LDS; parts meet through the caller's workspace: each part stores its sums,
// and the one that counts last adds them in part order, so that results do not
// depend on which part that is.
//
// What a row must not see cannot reach it: masked scores are replaced (not
// added to), places of the last tile past the length are cleared in V.  A
// value that is not finite in V would still turn the zero weight of another row of its
// tile into NaN, so rows whose result is not finite are computed again, one by
// one, over what they see (row_again).
#pragma once

#include "kv_dev.h"

namespace vq {

typedef __bf16 at_bf16x8 __attribute__((ext_vector_type(8)));
typedef float at_f32x4 __attribute__((ext_vector_type(4)));

constexpr int AT_NT = 256, AT_W = AT_NT / 64;
constexpr int AT_CNT = 2048;  // counters at the head of the workspace

struct AttnArgs {
    KvArgs c;
    const uint16_t* q;
    uint16_t* out;
    int64_t q_stride, out_stride;
    unsigned* cnt;
    float* part;
    int gqa, qgroups, splits, min_tiles, window, sinks;
    float scale;  // times log2 e
};

constexpr int at_qt_max(int D) { return D <= 128 ? 4 : 2; }
// Floats that one part leaves for one group of rows: sums, then {m, l} per row
__host__ __device__ constexpr size_t at_part_floats(int D, int qt) { return (size_t)qt * 16 * (D + 2); }
__host__ __device__ constexpr size_t at_lds_bytes(int D, int qt) {
    return (size_t)AT_W * qt * 16 * (D + 4) * 4 + (size_t)AT_W * qt * 16 * 8;
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

// One row computed on its own over the tokens that it sees: scores and weights
// by the thread of a token, sums by the thread of a dim.  Reached only by rows
// whose sums are not finite (values that are not, or pages that are missing).
template <int D, bool I8>
__device__ __forceinline__ void row_again(const AttnArgs& a, int b, int head, const uint16_t* q, uint16_t* o,
                                                    int p, float* lds) {
    const int tid = (int)threadIdx.x;
    const Sight sight{a.window, a.sinks};
    const int64_t cap = ((int64_t)a.c.width << a.c.tpl) * KV_TILE;
    float* w = lds;            // [AT_NT] weights of a chunk of tokens, -1: not seen
    float* acc = lds + AT_NT;  // [AT_NT]
    float* red = acc + AT_NT;  // [AT_W]
    float m = -__builtin_inff(), l = 0.0f, sum = 0.0f;
    bool bad = p >= cap;
#pragma unroll 1
    for (int pass = 0; pass < 2 && !bad; ++pass) {
        for (int64_t j0 = 0; j0 <= p; j0 += AT_NT) {
            // chunks between the first tokens and the window
            if (a.window != 0 && j0 >= a.sinks && j0 + AT_NT - 1 <= (int64_t)p - a.window) continue;
            const int64_t j64 = j0 + tid;
            const bool in = j64 <= p && sight.sees((int)j64, p);
            const int j = (int)(in ? j64 : p);
            const int tile = j / KV_TILE, t = j % KV_TILE;
            const int page = in ? kv_page(a.c, b, tile) : 0;
            float s = 0.0f;
            if (in && page < 0) bad = true;
            if (in && page >= 0) {
                const size_t at = kv_tile_at(a.c, page, head, tile), base = at * (KV_TILE * D);
#pragma unroll 1
                for (int c = 0; c < D / 8; ++c) {
                    for (int e = 0; e < 8; ++e) {
                        const float kv = I8 ? (float)((const int8_t*)a.c.k)[base + k_place<true>(t, c) + e]
                                            : bf16f(((const uint16_t*)a.c.k)[base + k_place<false>(t, c) + e]);
                        s = __builtin_fmaf(bf16f(q[8 * c + e]), kv, s);
                    }
                }
                if (I8) s *= a.c.ks[at * KV_TILE + t];
                s *= a.scale;
            }
            if (pass == 0) {
                if (in) m = fmaxf(m, s);
                continue;
            }
            const float e = in ? __builtin_amdgcn_exp2f(s - m) : -1.0f;
            if (in) l += e;
            __syncthreads();
            w[tid] = e;
            __syncthreads();
            const int d = tid % D;
#pragma unroll 1
            for (int i = tid / D; i < AT_NT; i += AT_NT / D) {
                if (w[i] == -1.0f) continue;  // (a weight is >= 0 or NaN)
                const int jt = (int)j0 + i, tl = jt / KV_TILE, tt = jt % KV_TILE;
                const size_t at = kv_tile_at(a.c, kv_page(a.c, b, tl), head, tl), base = at * (KV_TILE * D);
                const float vv = I8 ? (float)((const int8_t*)a.c.v)[base + v_place<true>(tt, d)] * a.c.vs[at * KV_TILE + tt]
                                    : bf16f(((const uint16_t*)a.c.v)[base + v_place<false>(tt, d)]);
                sum = __builtin_fmaf(w[i], vv, sum);
            }
        }
        // the maximum (first pass) and whether a page was missing, over the workgroup
        bad = __syncthreads_or(bad);
        if (pass == 0) {
            for (int off = 32; off > 0; off >>= 1) m = fmaxf(m, __shfl_xor(m, off, 64));
            if ((tid & 63) == 0) red[tid >> 6] = m;
            __syncthreads();
            m = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
        } else {
            for (int off = 32; off > 0; off >>= 1) l += __shfl_xor(l, off, 64);
            if ((tid & 63) == 0) red[tid >> 6] = l;
            acc[tid] = sum;
        }
        __syncthreads();
    }
    if (tid < D) {
        float v = __uint_as_float(0x7fc00000u);
        if (!bad) {
            v = 0.0f;
            for (int i = tid; i < AT_NT; i += D) v += acc[i];
            v /= red[0] + red[1] + red[2] + red[3];
        }
        o[tid] = f2bf(v);
    }
    __syncthreads();
}

template <int D, bool I8, int QT>
__global__ void __launch_bounds__(AT_NT)
attn_kernel(AttnArgs a) {
    constexpr int NKB = D / 32, NDB = D / 16, ROWS = QT * 16, ST = D + 4;
    constexpr int NK = I8 ? NKB : 2 * NKB, NV = I8 ? NDB / 2 : NDB;  // 16-byte loads of a lane per tile
    extern __shared__ __align__(16) float lds[];
    float* lo = lds;                       // [AT_W][ROWS][ST]
    float* lml = lds + AT_W * ROWS * ST;   // [AT_W][ROWS][2]
    __shared__ int last_part;
    __shared__ unsigned again[(ROWS + 31) / 32];

    const int tid = (int)threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int l16 = lane & 15, g = lane >> 4;
    int id = (int)blockIdx.x;
    const int split = id % a.splits;
    id /= a.splits;
    const int head = id % a.c.kvh;
    id /= a.c.kvh;
    const int b = id % a.c.batch, qg = id / a.c.batch;
    const KvSeq sq = kv_seq(a.c, b);
    const int rows = min(ROWS, sq.n * a.gqa - qg * ROWS);  // of this group
    if (rows <= 0) return;
    const int cap = (a.c.width << a.c.tpl) * KV_TILE;
    const int len = max(0, sq.len), hi = min(len, cap);
    const int pos0 = len - sq.n;  // position of the sequence's first row
    // the tiles that some row sees: those of the first tokens, then the window's
    int lo_t = 0, nsink = 0;
    if (a.window != 0) {
        const int from = max(0, pos0 + 1 > a.window ? pos0 + 1 - a.window : 0);
        nsink = (min(a.sinks, from) + KV_TILE - 1) / KV_TILE;
        lo_t = max(from / KV_TILE, nsink);
    }
    const int tiles = nsink + max(0, (hi + KV_TILE - 1) / KV_TILE - lo_t);
    const int want = min(a.splits, max(1, (tiles + a.min_tiles - 1) / a.min_tiles));
    const int per = max(1, (tiles + want - 1) / want);
    const int parts = max(1, (tiles + per - 1) / per);  // that have tiles
    if (split >= parts) return;
    const int t1 = min(tiles, (split + 1) * per);

    // Q as the operand with rows as its columns
    at_bf16x8 qf[QT][NKB];
    int pos[QT];  // position of the lane's row, -1: no row
#pragma unroll
    for (int qt = 0; qt < QT; ++qt) {
        const int rr = qt * 16 + l16, r = qg * ROWS + rr, i = r / a.gqa, hh = r - i * a.gqa;
        const bool ok = rr < rows;
        pos[qt] = ok ? pos0 + i : -1;
        const uint16_t* src = a.q + (size_t)(sq.row0 + (ok ? i : 0)) * a.q_stride + (size_t)(head * a.gqa + (ok ? hh : 0)) * D + 8 * g;
#pragma unroll
        for (int kb = 0; kb < NKB; ++kb) {
            u32x4 v = *(const u32x4*)(src + kb * 32);
            if (!ok) v = u32x4{0u, 0u, 0u, 0u};
            qf[qt][kb] = __builtin_bit_cast(at_bf16x8, v);
        }
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
    bool missing = len > cap;

    auto tile_of = [&](int v) { return v < nsink ? v : v - nsink + lo_t; };
    u32x4 kr[NK], vr[NV];
    float4 ksc[2], vsc[2];
    auto load_k = [&](int page, int tile) {
        const size_t at = kv_tile_at(a.c, page, head, tile);
        const u32x4* p = (const u32x4*)((const uint8_t*)a.c.k + at * (KV_TILE * D * (I8 ? 1 : 2))) + lane;
#pragma unroll
        for (int i = 0; i < NK; ++i) kr[i] = p[i * 64];
        if constexpr (I8) {
            const float4* s = (const float4*)(a.c.ks + at * KV_TILE + 8 * g);
            ksc[0] = s[0];
            ksc[1] = s[1];
        }
    };
    auto load_v = [&](int page, int tile) {
        const size_t at = kv_tile_at(a.c, page, head, tile);
        const u32x4* p = (const u32x4*)((const uint8_t*)a.c.v + at * (KV_TILE * D * (I8 ? 1 : 2))) + lane;
#pragma unroll
        for (int i = 0; i < NV; ++i) vr[i] = p[i * 64];
        if constexpr (I8) {
            const float4* s = (const float4*)(a.c.vs + at * KV_TILE + 8 * g);
            vsc[0] = s[0];
            vsc[1] = s[1];
        }
    };

    for (int v = split * per + wave; v < t1; v += AT_W) {
        const int tile = tile_of(v), page = kv_page(a.c, b, tile);
        if (page < 0) {
            missing = true;
            continue;
        }
        load_k(page, tile);
        load_v(page, tile);
        at_f32x4 S[QT][2];
#pragma unroll
        for (int qt = 0; qt < QT; ++qt) S[qt][0] = S[qt][1] = at_f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int kb = 0; kb < NKB; ++kb) {
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                at_bf16x8 k;
                if constexpr (I8) {
                    const u32x4 w = kr[(kb >> 1) * 2 + s];
                    k = kb & 1 ? codes_bf16(w.z, w.w) : codes_bf16(w.x, w.y);
                } else {
                    k = __builtin_bit_cast(at_bf16x8, kr[kb * 2 + s]);
                }
#pragma unroll
                for (int qt = 0; qt < QT; ++qt)
                    S[qt][s] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k, qf[qt][kb], S[qt][s], 0, 0, 0);
            }
        }
        // scores, by token of the lane's eight; tiles that some row does not see whole are masked
        const int j0 = tile * KV_TILE, jl = j0 + 8 * g;
        const bool whole = j0 + KV_TILE - 1 <= pos0 &&
                           (a.window == 0 || j0 > len - 1 - a.window || j0 + KV_TILE <= a.sinks);
        at_bf16x8 ph[QT], pl[QT];
        const float* kscale = (const float*)ksc;
        const float* vscale = (const float*)vsc;
#pragma unroll
        for (int qt = 0; qt < QT; ++qt) {
            float x[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                x[e] = S[qt][e >> 2][e & 3] * a.scale;
                if constexpr (I8) x[e] *= kscale[e];
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
    }

    // the waves meet
#pragma unroll
    for (int qt = 0; qt < QT; ++qt) {
        const int row = wave * ROWS + qt * 16 + l16;
        const float lt = sum_over_groups(l[qt]);
        if (g == 0) {
            lml[2 * row] = m[qt];
            lml[2 * row + 1] = missing ? __uint_as_float(0x7fc00000u) : lt;
        }
#pragma unroll
        for (int db = 0; db < NDB; ++db) *(at_f32x4*)(lo + row * ST + 16 * db + 4 * g) = O[qt][db];
    }
    if (tid < (ROWS + 31) / 32) again[tid] = 0u;
    __syncthreads();

    const int rec = (qg * a.c.batch + b) * a.c.kvh + head;
    const size_t floats = at_part_floats(D, QT);
    // a row's result, or what its waves or parts have found so far
    auto store = [&](int rr, int d, at_f32x4 o, float lt) {
        const int r = qg * ROWS + rr, i = r / a.gqa, hh = r - i * a.gqa, p = pos0 + i;
        const float inv = 1.0f / lt;
        o = o * inv;
        if (p < 0) o = at_f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        // (0 * x is NaN where x is not finite)
        else if (!(o[0] * 0.0f + o[1] * 0.0f + o[2] * 0.0f + o[3] * 0.0f == 0.0f)) atomicOr(&again[rr >> 5], 1u << (rr & 31));
        *(u32x2*)(a.out + (size_t)(sq.row0 + i) * a.out_stride + (size_t)(head * a.gqa + hh) * D + d) =
            u32x2{f2bf2(o[0], o[1]), f2bf2(o[2], o[3])};
    };
    for (int i = tid; i < rows * (D / 4); i += AT_NT) {
        const int rr = i / (D / 4), d = i % (D / 4) * 4;
        float M = lml[2 * rr];
#pragma unroll
        for (int w = 1; w < AT_W; ++w) M = fmaxf(M, lml[2 * (w * ROWS + rr)]);
        at_f32x4 o = {0.0f, 0.0f, 0.0f, 0.0f};
        float lt = 0.0f;
#pragma unroll
        for (int w = 0; w < AT_W; ++w) {
            const float f = part_weight(lml[2 * (w * ROWS + rr)], M), lw = lml[2 * (w * ROWS + rr) + 1];
            o += *(const at_f32x4*)(lo + (w * ROWS + rr) * ST + d) * f;
            lt += lw == lw ? lw * f : lw;
        }
        if (parts == 1) {
            store(rr, d, o, lt);
        } else {
            float* pr = a.part + ((size_t)rec * a.splits + split) * floats;
            *(at_f32x4*)(pr + rr * D + d) = o;
            if (d == 0) *(float2*)(pr + ROWS * D + 2 * rr) = make_float2(M, lt);
        }
    }
    if (parts > 1) {
        __threadfence();
        __syncthreads();
        if (tid == 0) {
            const unsigned old = __hip_atomic_fetch_add(a.cnt + rec, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            last_part = old == (unsigned)(parts - 1);
            if (last_part) __hip_atomic_store(a.cnt + rec, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        }
        __syncthreads();
        if (!last_part) return;
        __threadfence();
        const float* pr = a.part + (size_t)rec * a.splits * floats;
        for (int i = tid; i < rows * (D / 4); i += AT_NT) {
            const int rr = i / (D / 4), d = i % (D / 4) * 4;
            float M = -__builtin_inff(), lt = 0.0f;
            at_f32x4 o = {0.0f, 0.0f, 0.0f, 0.0f};
            for (int s = 0; s < parts; ++s) M = fmaxf(M, pr[s * floats + ROWS * D + 2 * rr]);
            for (int s = 0; s < parts; ++s) {
                const float2 ml = *(const float2*)(pr + s * floats + ROWS * D + 2 * rr);
                const float f = part_weight(ml.x, M);
                o += *(const at_f32x4*)(pr + s * floats + rr * D + d) * f;
                lt += ml.y == ml.y ? ml.y * f : ml.y;
            }
            store(rr, d, o, lt);
        }
    }
    __syncthreads();
    for (int rr = 0; rr < rows; ++rr) {
        if (!((again[rr >> 5] >> (rr & 31)) & 1u)) continue;
        const int r = qg * ROWS + rr, i = r / a.gqa, hh = r - i * a.gqa;
        const size_t row = (size_t)sq.row0 + i, h = (size_t)(head * a.gqa + hh) * D;
        row_again<D, I8>(a, b, head, a.q + row * a.q_stride + h, a.out + row * a.out_stride + h, pos0 + i, lds);
    }
}

template <bool I8>
inline const void* attn_fn(int D, int qt) {
    switch (D * 8 + qt) {
        case 64 * 8 + 1: return (const void*)attn_kernel<64, I8, 1>;
        case 64 * 8 + 2: return (const void*)attn_kernel<64, I8, 2>;
        case 64 * 8 + 3: return (const void*)attn_kernel<64, I8, 3>;
        case 64 * 8 + 4: return (const void*)attn_kernel<64, I8, 4>;
        case 128 * 8 + 1: return (const void*)attn_kernel<128, I8, 1>;
        case 128 * 8 + 2: return (const void*)attn_kernel<128, I8, 2>;
        case 128 * 8 + 3: return (const void*)attn_kernel<128, I8, 3>;
        case 128 * 8 + 4: return (const void*)attn_kernel<128, I8, 4>;
        case 256 * 8 + 1: return (const void*)attn_kernel<256, I8, 1>;
        case 256 * 8 + 2: return (const void*)attn_kernel<256, I8, 2>;
        default: return nullptr;
    }
}

}  // namespace vq
