// Rows into and out of the paged key/value cache.
//
// append: row r of a sequence is token p = len - n + r.  For theta > 0 its q and
// k are rotated by a_i = p theta^(-2i/D): (x_i, x_(i+D/2)) -> (x_i cos a_i -
// x_(i+D/2) sin a_i, x_(i+D/2) cos a_i + x_i sin a_i).  Angles grow with p (10^5
// and more) while cos and sin need them to a fraction of 2 pi, which 32 bits do
// not hold, so angles, cos, sin and the two products are 64-bit; a row has D/2
// angles that all its heads share, so they are computed once per workgroup into
// LDS while the row's values are in flight.  The result is rounded to fp32
// and from there to bf16 (what attention reads; 2^-16 of a step more than one
// rounding) and, for int8 caches, quantized from that bf16 row with one
// scale, by the activation quantizer's exact RNE(x / s).
//
// Work: a workgroup per row and 256 threads of units; a unit (one head's q, k or
// v row) is D / 16 threads with octets o and o + D/16, the pair that rotation
// mixes.  K octets are contiguous in the tile's order; V is stored token by token
// with 2-byte stores (1-byte for int8), since 8 tokens of a dim share 16 bytes.
// Bound by latency at a decode step's sizes (one row of 20 + 4 + 4 heads of 128: 2.7
// us, of which 1.5 are the dispatch), by the small V stores at a batch's (512 rows of
// 64 sequences into int8 5.9 us).  FP4 caches have a kernel of their own (kv_append4_kernel).

#include "kv_host.h"

namespace vq {

constexpr int KA_NT = 256;

struct AppendArgs {
    KvArgs c;
    const uint16_t* k;
    const uint16_t* v;
    const uint16_t* q;
    uint16_t* qo;
    int64_t kv_stride, q_stride, qo_stride;
    int heads, ub;  // workgroups per row (FP4: per octet of tokens)
    int octets;     // FP4: that a sequence's rows can touch
    double log2_theta;
};

__device__ __forceinline__ void to_f32(const u32x4& v, float* f) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        f[2 * i] = bf16f(w[i] & 0xffffu);
        f[2 * i + 1] = bf16f(w[i] >> 16);
    }
}
__device__ __forceinline__ u32x4 to_bf16(const float* f) {
    return u32x4{f2bf2(f[0], f[1]), f2bf2(f[2], f[3]), f2bf2(f[4], f[5]), f2bf2(f[6], f[7])};
}

// Largest of a value over the D / 16 (4, 8 or 16) consecutive lanes of a unit
template <int L>
__device__ __forceinline__ float unit_max(float v) {
    v = fmaxf(v, dpp_f<DPP_SWAP1>(v));
    v = fmaxf(v, dpp_f<DPP_SWAP2>(v));
    if constexpr (L >= 8) v = fmaxf(v, dpp_f<DPP_HALF_MIRROR>(v));
    if constexpr (L >= 16) v = fmaxf(v, dpp_f<DPP_MIRROR>(v));
    return v;
}

// FP4: the exponent of a block of keys whose largest magnitude is m, 2^e the least
// power with m <= 7 * 2^e (a value over 6 becomes 6, which is as near as 8 would be)
__device__ __forceinline__ int fp4_exponent(float m) {
    const uint32_t u = __float_as_uint(m);
    const int e = (int)(u >> 23) - 129 + ((u & 0x7fffffu) > 0x600000u ? 1 : 0);
    return min(125, max(-125, e));
}
// Codes of 8 values times f, rounded to nearest even and at most 6 in magnitude
__device__ __forceinline__ uint32_t fp4_codes(const float* x, float f) {
    uint32_t w = 0;
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[0] * f, x[1] * f, 1.0f, 0);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[2] * f, x[3] * f, 1.0f, 1);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[4] * f, x[5] * f, 1.0f, 2);
    return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[6] * f, x[7] * f, 1.0f, 3);
}

template <int D, bool I8, bool ROPE>
__global__ void __launch_bounds__(KA_NT)
kv_append_kernel(AppendArgs a) {
    constexpr int TPU = D / 16, UPB = KA_NT / TPU;
    __shared__ double cs[D / 2], sn[D / 2];
    const int row_id = (int)blockIdx.x / a.ub, ub = (int)blockIdx.x % a.ub;
    const int b = row_id / a.c.max_rows, r = row_id % a.c.max_rows;
    const KvSeq s = kv_seq(a.c, b);
    if (r >= s.n) return;
    const int64_t pos64 = (int64_t)s.len - s.n + r;
    if (pos64 < 0) return;
    const int pos = (int)pos64;
    const int tid = (int)threadIdx.x;
    const int unit = ub * UPB + tid / TPU, o = tid % TPU;
    const int nq = ROPE && a.q != nullptr ? a.heads : 0;
    const bool is_q = unit < nq, is_k = !is_q && unit < nq + a.c.kvh, live = unit < nq + 2 * a.c.kvh;
    const int head = is_q ? unit : (unit - nq) % a.c.kvh;
    const size_t row = (size_t)s.row0 + r;
    u32x4 x0 = {0u, 0u, 0u, 0u}, x1 = x0;
    if (live) {
        const uint16_t* src = is_q ? a.q + row * a.q_stride : (is_k ? a.k : a.v) + row * a.kv_stride;
        src += (size_t)head * D + 8 * o;
        x0 = *(const u32x4*)src;
        x1 = *(const u32x4*)(src + D / 2);
    }
    if constexpr (ROPE) {
        if (tid < D / 2) {
            const double f = exp2(-(double)tid * (2.0 / D) * a.log2_theta);
            double sv, cv;
            sincos((double)pos * f, &sv, &cv);
            cs[tid] = cv;
            sn[tid] = sv;
        }
        __syncthreads();
        if (is_q || is_k) {
            float f0[8], f1[8];
            to_f32(x0, f0);
            to_f32(x1, f1);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const double c = cs[8 * o + j], n = sn[8 * o + j], u = (double)f0[j], w = (double)f1[j];
                f0[j] = (float)(u * c - w * n);
                f1[j] = (float)(w * c + u * n);
            }
            x0 = to_bf16(f0);
            x1 = to_bf16(f1);
        }
    }
    uint32_t q0[2], q1[2];
    float scale = 0.0f;
    if constexpr (I8) {
        float f0[8], f1[8];
        to_f32(x0, f0);
        to_f32(x1, f1);
        float amax = 0.0f, sum = 0.0f;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            amax = fmaxf(amax, fmaxf(fabsf(f0[j]), fabsf(f1[j])));
            sum += f0[j] * 0.0f + f1[j] * 0.0f;  // NaN where a value is not finite
        }
        amax = unit_max<TPU>(amax);
        const bool finite = unit_max<TPU>(sum == sum ? 0.0f : 1.0f) == 0.0f;
        float rc;
        group_scale(amax, scale, rc);
        uint32_t t[16];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            t[j] = qbits(f0[j], scale, rc);
            t[8 + j] = qbits(f1[j], scale, rc);
        }
        q0[0] = bytes4(t[0], t[1], t[2], t[3]);
        q0[1] = bytes4(t[4], t[5], t[6], t[7]);
        q1[0] = bytes4(t[8], t[9], t[10], t[11]);
        q1[1] = bytes4(t[12], t[13], t[14], t[15]);
        if (!finite) scale = __uint_as_float(0x7fc00000u);  // the row reads back as NaN
    }
    if (!live) return;
    if (is_q) {
        uint16_t* dst = a.qo + row * a.qo_stride + (size_t)head * D + 8 * o;
        *(u32x4*)dst = x0;
        *(u32x4*)(dst + D / 2) = x1;
        return;
    }
    const int tile = pos / KV_TILE, t = pos % KV_TILE;
    const int page = kv_page(a.c, b, tile);
    if (page < 0) return;
    const size_t at = kv_tile_at(a.c, page, head, tile), base = at * (KV_TILE * D);
    if (is_k) {
        if constexpr (I8) {
            int8_t* p = (int8_t*)a.c.k + base;
            *(u32x2*)(p + k_place<true>(t, o)) = u32x2{q0[0], q0[1]};
            *(u32x2*)(p + k_place<true>(t, o + TPU)) = u32x2{q1[0], q1[1]};
            if (o == 0) a.c.ks[at * KV_TILE + t] = scale;
        } else {
            uint16_t* p = (uint16_t*)a.c.k + base;
            *(u32x4*)(p + k_place<false>(t, o)) = x0;
            *(u32x4*)(p + k_place<false>(t, o + TPU)) = x1;
        }
        return;
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        if constexpr (I8) {
            int8_t* p = (int8_t*)a.c.v + base;
            p[v_place<true>(t, 8 * o + j)] = (int8_t)(q0[j >> 2] >> (8 * (j & 3)));
            p[v_place<true>(t, D / 2 + 8 * o + j)] = (int8_t)(q1[j >> 2] >> (8 * (j & 3)));
        } else {
            const uint32_t w0[4] = {x0.x, x0.y, x0.z, x0.w}, w1[4] = {x1.x, x1.y, x1.z, x1.w};
            uint16_t* p = (uint16_t*)a.c.v + base;
            p[v_place<false>(t, 8 * o + j)] = (uint16_t)(w0[j >> 1] >> (16 * (j & 1)));
            p[v_place<false>(t, D / 2 + 8 * o + j)] = (uint16_t)(w1[j >> 1] >> (16 * (j & 1)));
        }
    }
    if (I8 && o == 0) a.c.vs[at * KV_TILE + t] = scale;
}

// FP4: two tokens of a value share a byte and eight a word, so a workgroup takes the
// rows of one octet of tokens (one row of a decode step, eight of a prompt) and stores its
// words whole, those of an octet that the call does not fill with what they held of the
// other tokens (flipping their bits by atomics took 8.6 us for one row, this 3.5).
// The angles of all rows are in LDS before the first: those of the first row and of one
// step by sincos, each further row's by the sum of angles (4 products of 64 bits).  A
// row's values are in flight while the one before is rounded.  9700 rows of 20 + 4 + 4 heads
// of 128 in 33.5 us (124 MB): 13 are VALU issue, two thirds of it the rotation's, and waves wait
// 57 % of their time, four to a SIMD (101 registers; 1220 octets are a round of 1024 workgroups and
// a fifth of another).  Not more rows in flight, nor whole tiles to one XCD made a difference.
template <int D, bool ROPE>
__global__ void __launch_bounds__(KA_NT)
kv_append4_kernel(AppendArgs a) {
    constexpr int TPU = D / 16, UPB = KA_NT / TPU;
    __shared__ double cs[8][D / 2], sn[8][D / 2];  // dim 8 o + j at [TPU j + o]: neighbouring threads read neighbours
    auto turn_at = [](int d) { return TPU * (d % 8) + d / 8; };
    int id = (int)blockIdx.x;
    const int ub = id % a.ub;
    id /= a.ub;
    const int b = id / a.octets, oc = id % a.octets;
    const KvSeq s = kv_seq(a.c, b);
    const int64_t p0 = (int64_t)s.len - s.n;  // position of row 0
    const int64_t from = p0 < 0 ? 0 : p0;
    const int64_t lo64 = (from / 8 + oc) * 8;
    if (s.n == 0 || lo64 >= s.len) return;
    const int lo = (int)lo64;
    const int t0 = (int)(from > lo64 ? from - lo64 : 0), t1 = min(8, s.len - lo);  // rows of the octet
    const int tid = (int)threadIdx.x;
    const int unit = ub * UPB + tid / TPU, o = tid % TPU;
    const int nq = ROPE && a.q != nullptr ? a.heads : 0;
    const bool is_q = unit < nq, is_k = !is_q && unit < nq + a.c.kvh, live = unit < nq + 2 * a.c.kvh;
    const int head = is_q ? unit : (unit - nq) % a.c.kvh;
    const size_t row0 = (size_t)(s.row0 + ((int64_t)lo - p0));  // row of the octet's token 0
    const int64_t stride = is_q ? a.q_stride : a.kv_stride;
    const uint16_t* src = (is_q ? a.q : is_k ? a.k : a.v) + (size_t)head * D + 8 * o;
    u32x4 n0, n1;
    auto fetch = [&](int t) {  // (past the last row: that row, and for threads past the units a value's)
        const uint16_t* p = src + (row0 + min(t, t1 - 1)) * stride;
        n0 = *(const u32x4*)p;
        n1 = *(const u32x4*)(p + D / 2);
    };
    fetch(t0);
    const int tile = lo / KV_TILE, tt = lo % KV_TILE;
    const int page = is_q ? -1 : kv_page(a.c, b, tile);
    const size_t at = page >= 0 ? kv_tile_at(a.c, page, head, tile) : 0;
    uint8_t* const kt = (uint8_t*)a.c.k + at * (KV_TILE * D / 2);
    uint8_t* const vt = (uint8_t*)a.c.v + at * (KV_TILE * D / 2);
    const bool is_v = live && !is_q && !is_k && page >= 0, full = t0 == 0 && t1 == 8;
    uint32_t words[16], old[16];
    auto word_at = [&](int j) { return (uint32_t*)(vt + v4_place(tt, (j < 8 ? 8 * o : D / 2 + 8 * o - 8) + j)); };
#pragma unroll
    for (int j = 0; j < 16; ++j) {
        words[j] = 0u;
        old[j] = is_v && !full ? *word_at(j) : 0u;
    }
    if constexpr (ROPE) {
        double cv = 0.0, sv = 0.0;
        const bool several = t1 - t0 > 1;
        if (tid < (several ? D : D / 2)) {  // the upper half: one step
            const int d = tid % (D / 2);
            const double f = exp2(-(double)d * (2.0 / D) * a.log2_theta);
            sincos(tid < D / 2 ? (double)(lo + t0) * f : f, &sv, &cv);
            if (tid >= D / 2) {  // (in the last row's place until the barriers; a row alone may be that one)
                cs[7][d] = cv;
                sn[7][d] = sv;
            }
        }
        double c1 = 0.0, s1 = 0.0;
        if (several) {
            __syncthreads();
            if (tid < D / 2) {
                c1 = cs[7][tid];
                s1 = sn[7][tid];
            }
            __syncthreads();
        }
        if (tid < D / 2) {
            for (int t = t0; t < t1; ++t) {
                cs[t][turn_at(tid)] = cv;
                sn[t][turn_at(tid)] = sv;
                const double c = cv * c1 - sv * s1;
                sv = sv * c1 + cv * s1;
                cv = c;
            }
        }
        __syncthreads();
    }
    for (int t = t0; t < t1; ++t) {
        u32x4 x0 = n0, x1 = n1;
        fetch(t + 1);
        float f0[8], f1[8];
        to_f32(x0, f0);
        to_f32(x1, f1);
        if (ROPE && (is_q || is_k)) {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const double c = cs[t][TPU * j + o], n = sn[t][TPU * j + o], u = (double)f0[j], w = (double)f1[j];
                f0[j] = (float)(u * c - w * n);
                f1[j] = (float)(w * c + u * n);
            }
            x0 = to_bf16(f0);
            x1 = to_bf16(f1);
            if (is_q) {
                uint16_t* dst = a.qo + (row0 + t) * a.qo_stride + (size_t)head * D + 8 * o;
                *(u32x4*)dst = x0;
                *(u32x4*)(dst + D / 2) = x1;
            }
            to_f32(x0, f0);
            to_f32(x1, f1);
        }
        if (is_q) continue;
        // blocks of 32 dims are four lanes' octets, on either side of the row's middle
        float m0 = 0.0f, m1 = 0.0f, bad0 = 0.0f, bad1 = 0.0f;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            m0 = fmaxf(m0, fabsf(f0[j]));
            m1 = fmaxf(m1, fabsf(f1[j]));
            bad0 += f0[j] * 0.0f;  // NaN where a value is not finite
            bad1 += f1[j] * 0.0f;
        }
        m0 = group_max<4>(m0);
        m1 = group_max<4>(m1);
        bad0 = group_max<4>(bad0 == bad0 ? 0.0f : 1.0f);
        bad1 = group_max<4>(bad1 == bad1 ? 0.0f : 1.0f);
        if (is_k && page >= 0) {
            const int e0 = fp4_exponent(m0), e1 = fp4_exponent(m1);
            *(uint32_t*)(kt + k4_place<D>(tt + t, o)) = fp4_codes(f0, __uint_as_float((uint32_t)(127 - e0) << 23));
            *(uint32_t*)(kt + k4_place<D>(tt + t, o + TPU)) = fp4_codes(f1, __uint_as_float((uint32_t)(127 - e1) << 23));
            if (o % 4 == 0) {
                uint8_t* const ex = (uint8_t*)a.c.ks + at * D;
                ex[k4_exp_place<D>(tt + t, o / 4)] = (uint8_t)(bad0 != 0.0f ? 255 : e0 + 127);
                ex[k4_exp_place<D>(tt + t, (o + TPU) / 4)] = (uint8_t)(bad1 != 0.0f ? 255 : e1 + 127);
            }
        }
        const float amax = unit_max<TPU>(fmaxf(m0, m1)), bad = unit_max<TPU>(fmaxf(bad0, bad1));
        if (is_v) {
            const float scale = fmaxf(amax / 6.0f, 1e-8f), rc = __builtin_amdgcn_rcpf(scale);
            // the quotient by the hardware's reciprocal and one step of correction: the code
            // equals that of the IEEE quotient for every pair of a bf16 value and a row's
            // largest (a test goes through all of their mantissas)
            auto quotient = [&](float x) {
                const float y = x * rc;
                return __builtin_fmaf(rc, __builtin_fmaf(-y, scale, x), y);
            };
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                f0[j] = quotient(f0[j]);
                f1[j] = quotient(f1[j]);
            }
            const uint32_t c0 = fp4_codes(f0, 1.0f), c1 = fp4_codes(f1, 1.0f);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                words[j] |= ((c0 >> (4 * j)) & 15u) << (4 * t);
                words[8 + j] |= ((c1 >> (4 * j)) & 15u) << (4 * t);
            }
            if (o == 0) a.c.vs[at * KV_TILE + tt + t] = bad != 0.0f ? __uint_as_float(0x7fc00000u) : scale;
        }
    }
    if (!is_v) return;
    const uint32_t mine = (t1 == 8 ? 0xffffffffu : (1u << (4 * t1)) - 1u) & (0xffffffffu << (4 * t0));
#pragma unroll
    for (int j = 0; j < 16; ++j) *word_at(j) = full ? words[j] : (old[j] & ~mine) | words[j];
}

// read: a workgroup per tile of 32 tokens, pool (K, V) and head, of 64 dims two heads
// whose loads are in flight together (a workgroup's chain of length, page and tile
// takes longer than moving so small a tile).  K octets go straight to their rows; V turns
// through LDS (8 tokens of a dim arrive together).  Threads follow the output rows, so
// that each wave stores whole lines.
struct ReadArgs {
    KvArgs c;
    uint16_t* ko;
    uint16_t* vo;
    int tiles;   // tiles that a sequence's rows can touch
    int groups;  // of heads
};

// (8 heads of 64 dims, int8, 18000 rows of 8 sequences: 1 head 16.2 us, 2 13.0, 4 12.6; 4 rows of
// 16 sequences 3.1 / 3.4 / 4.3; 4 heads of 128 dims, 4096 rows of 64: 1 head 4.3, 4 7.6)
constexpr int kr_heads(int D) { return D == 64 ? 2 : 1; }

template <int D, int KT>
__global__ void __launch_bounds__(KA_NT)
kv_read_kernel(ReadArgs a) {
    constexpr bool I8 = KT == VIPER_KV_INT8, F4 = KT == VIPER_KV_FP4;
    constexpr int OPR = D / 8, HG = kr_heads(D);                 // octets of a row, heads
    constexpr int PT = KV_TILE * OPR / KA_NT;                    // octets of a head and thread
    __shared__ __align__(16) uint16_t lv[HG][KV_TILE][D + 8];
    int id = (int)blockIdx.x;
    const int side = id & 1;
    id >>= 1;
    const int head0 = id % a.groups * HG;
    id /= a.groups;
    const int b = id / a.tiles;
    const KvSeq s = kv_seq(a.c, b);
    if (s.n == 0) return;
    const int64_t p0 = (int64_t)s.len - s.n;  // position of row 0
    const int64_t tile0 = (p0 < 0 ? 0 : p0) / KV_TILE, tile64 = tile0 + id % a.tiles;
    if (tile64 * KV_TILE >= s.len) return;
    const int tile = (int)tile64, tid = (int)threadIdx.x;
    const int page = kv_page_uniform(a.c, b, tile);
    const int heads = min(HG, a.c.kvh - head0);
    const float* scales = side == 0 ? a.c.ks : a.c.vs;
    const void* pool = side == 0 ? a.c.k : a.c.v;
    uint16_t* out = side == 0 ? a.ko : a.vo;
    // octet i of a thread: K (token, octet of the row), V (8 tokens, dim)
    u32x4 x[HG][PT];
#pragma unroll
    for (int h = 0; h < HG; ++h) {
        if (h >= heads || page < 0) continue;
        const size_t base = kv_tile_at(a.c, page, head0 + h, tile) * (KV_TILE * D);
#pragma unroll
        for (int k = 0; k < PT; ++k) {
            const int i = tid + k * KA_NT;
            if constexpr (F4) {
                const int e = side == 0 ? k4_place<D>(i / OPR, i % OPR) : v4_place(8 * (i / D), i % D);
                x[h][k] = u32x4{*(const uint32_t*)((const uint8_t*)pool + base / 2 + e), 0u, 0u, 0u};
                continue;
            }
            const int e = side == 0 ? k_place<I8>(i / OPR, i % OPR) : v_place<I8>(8 * (i / D), i % D);
            if constexpr (I8) {
                const u32x2 w = *(const u32x2*)((const int8_t*)pool + base + e);
                x[h][k] = u32x4{w.x, w.y, 0u, 0u};
            } else {
                x[h][k] = *(const u32x4*)((const uint16_t*)pool + base + e);
            }
        }
    }
    auto store = [&](int h, int t, int c, const u32x4& v) {
        const int64_t r = (int64_t)tile * KV_TILE + t - p0;
        if (r >= 0 && r < s.n) *(u32x4*)(out + ((size_t)(s.row0 + r) * a.c.kvh + head0 + h) * D + 8 * c) = v;
    };
#pragma unroll
    for (int h = 0; h < HG; ++h) {
        if (h >= heads) continue;
        const float* sc = nullptr;
        const uint8_t* ex = nullptr;
        if ((I8 || F4) && page >= 0) {
            const size_t at = kv_tile_at(a.c, page, head0 + h, tile);
            sc = scales + at * KV_TILE;
            ex = (const uint8_t*)a.c.ks + at * D;
        }
#pragma unroll
        for (int k = 0; k < PT; ++k) {
            const int i = tid + k * KA_NT;
            if (page < 0) {
                store(h, i / OPR, i % OPR, u32x4{0u, 0u, 0u, 0u});
                continue;
            }
            u32x4 v = x[h][k];
            if constexpr (I8) {
                float y[8];
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    y[j] = (float)(int8_t)((j < 4 ? v.x : v.y) >> (8 * (j & 3))) * (side == 0 ? sc[i / OPR] : sc[8 * (i / D) + j]);
                v = to_bf16(y);
            } else if constexpr (F4) {
                if (side == 0) {
                    v = fp4_bf16(v.x, fp4_power(ex[k4_exp_place<D>(i / OPR, i % OPR / 4)]));
                } else {
                    float y[8];
                    fp4_f32(v.x, 1.0f, y);
#pragma unroll
                    for (int j = 0; j < 8; ++j) y[j] *= sc[8 * (i / D) + j];
                    v = to_bf16(y);
                }
            }
            if (side == 0) {
                store(h, i / OPR, i % OPR, v);
            } else {
                const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                for (int j = 0; j < 8; ++j) lv[h][8 * (i / D) + j][i % D] = (uint16_t)(w[j >> 1] >> (16 * (j & 1)));
            }
        }
    }
    if (side == 0 || page < 0) return;
    __syncthreads();
#pragma unroll
    for (int h = 0; h < HG; ++h) {
        if (h >= heads) continue;
#pragma unroll
        for (int k = 0; k < PT; ++k) {
            const int i = tid + k * KA_NT;
            store(h, i / OPR, i % OPR, *(const u32x4*)&lv[h][i / OPR][8 * (i % OPR)]);
        }
    }
}

template <int D>
static const void* append_fn(bool i8, bool rope) {
    if (i8) return rope ? (const void*)kv_append_kernel<D, true, true> : (const void*)kv_append_kernel<D, true, false>;
    return rope ? (const void*)kv_append_kernel<D, false, true> : (const void*)kv_append_kernel<D, false, false>;
}
template <int D>
static const void* append4_fn(bool rope) {
    return rope ? (const void*)kv_append4_kernel<D, true> : (const void*)kv_append4_kernel<D, false>;
}
template <int D>
static const void* read_fn(int kv) {
    return kv == VIPER_KV_INT8  ? (const void*)kv_read_kernel<D, VIPER_KV_INT8>
           : kv == VIPER_KV_FP4 ? (const void*)kv_read_kernel<D, VIPER_KV_FP4>
                                : (const void*)kv_read_kernel<D, VIPER_KV_BF16>;
}

constexpr int64_t GRID_MAX = (1 << 24) - 1;  // workgroups of 256 threads: under 2^32 threads
// No sequence has more rows than the tensors hold: what the grid is sized by (max_rows may be any bound)
static int rows_most(const viper_kv_batch* b) { return b->max_rows < b->total_rows ? b->max_rows : b->total_rows; }

}  // namespace vq

extern "C" int viper_hip_kv_append(const viper_kv_cache* cache, const viper_kv_batch* batch, const void* k_bf16,
                                   const void* v_bf16, int64_t kv_stride, const void* q_bf16, int64_t q_stride, int heads,
                                   void* q_out_bf16, int64_t q_out_stride, double rope_theta, void* stream) {
    using namespace vq;
    int rc = kv_check(cache, batch);
    if (rc != VIPER_OK) return rc;
    const int D = cache->head_dim;
    const int64_t width = (int64_t)cache->kv_heads * D;
    if (bad_rows(k_bf16, kv_stride, width) || bad_rows(v_bf16, kv_stride, width)) return VIPER_INVALID_ARGUMENT;
    if (!(rope_theta >= 0.0) || rope_theta > 1e30 || (rope_theta > 0.0 && rope_theta < 1.0)) return VIPER_INVALID_ARGUMENT;
    const bool rope = rope_theta > 0.0;
    if (q_bf16 != nullptr) {
        if (!rope || heads <= 0 || heads > 65536) return VIPER_INVALID_ARGUMENT;
        if (bad_rows(q_bf16, q_stride, (int64_t)heads * D) || bad_rows(q_out_bf16, q_out_stride, (int64_t)heads * D))
            return VIPER_INVALID_ARGUMENT;
    } else if (q_out_bf16 != nullptr) {
        return VIPER_INVALID_ARGUMENT;
    }
    if (batch->total_rows == 0) return VIPER_OK;
    if (q_bf16 != nullptr) {  // q_out may be q, and nothing else that other workgroups read
        const int64_t n = batch->total_rows, qw = (int64_t)heads * D;
        if ((q_out_bf16 != q_bf16 || (q_out_stride != q_stride && n > 1)) &&
            rows_meet(q_bf16, q_stride, qw, q_out_bf16, q_out_stride, qw, n))
            return VIPER_INVALID_ARGUMENT;
        if (rows_meet(k_bf16, kv_stride, width, q_out_bf16, q_out_stride, qw, n) ||
            rows_meet(v_bf16, kv_stride, width, q_out_bf16, q_out_stride, qw, n))
            return VIPER_INVALID_ARGUMENT;
    }
    AppendArgs a;
    a.c = kv_args(cache, batch);
    a.k = (const uint16_t*)k_bf16;
    a.v = (const uint16_t*)v_bf16;
    a.q = (const uint16_t*)q_bf16;
    a.qo = (uint16_t*)q_out_bf16;
    a.kv_stride = kv_stride;
    a.q_stride = q_stride;
    a.qo_stride = q_out_stride;
    a.heads = q_bf16 != nullptr ? heads : 0;
    a.log2_theta = rope ? __builtin_log2(rope_theta) : 0.0;
    const int units = a.heads + 2 * cache->kv_heads, upb = KA_NT / (D / 16);
    a.ub = (units + upb - 1) / upb;
    a.c.max_rows = rows_most(batch);
    const bool i8 = cache->kv_type == VIPER_KV_INT8, f4 = cache->kv_type == VIPER_KV_FP4;
    a.octets = (int)(((int64_t)a.c.max_rows + 6) / 8 + 1);
    const int64_t grid = (int64_t)batch->batch * (f4 ? a.octets : a.c.max_rows) * a.ub;
    if (grid > GRID_MAX) return VIPER_INVALID_ARGUMENT;
    const void* fn = f4 ? (D == 64 ? append4_fn<64>(rope) : D == 128 ? append4_fn<128>(rope) : append4_fn<256>(rope))
                     : D == 64 ? append_fn<64>(i8, rope) : D == 128 ? append_fn<128>(i8, rope) : append_fn<256>(i8, rope);
    void* args[] = {&a};
    launch(fn, (unsigned)grid, KA_NT, 0, (hipStream_t)stream, args);
    return status_of(hipGetLastError());
}

extern "C" int viper_hip_kv_read(const viper_kv_cache* cache, const viper_kv_batch* batch, void* k_out_bf16,
                                 void* v_out_bf16, void* stream) {
    using namespace vq;
    int rc = kv_check(cache, batch);
    if (rc != VIPER_OK) return rc;
    if (k_out_bf16 == nullptr || v_out_bf16 == nullptr || misaligned(k_out_bf16, 16) || misaligned(v_out_bf16, 16))
        return VIPER_INVALID_ARGUMENT;
    if (batch->total_rows == 0) return VIPER_OK;
    const int64_t row = (int64_t)cache->kv_heads * cache->head_dim;
    if (rows_meet(k_out_bf16, row, row, v_out_bf16, row, row, batch->total_rows)) return VIPER_INVALID_ARGUMENT;
    ReadArgs a;
    a.c = kv_args(cache, batch);
    a.ko = (uint16_t*)k_out_bf16;
    a.vo = (uint16_t*)v_out_bf16;
    a.c.max_rows = rows_most(batch);
    const int64_t tiles = ((int64_t)a.c.max_rows + KV_TILE - 2) / KV_TILE + 1;
    a.tiles = (int)tiles;
    a.groups = (cache->kv_heads + kr_heads(cache->head_dim) - 1) / kr_heads(cache->head_dim);
    const int64_t grid = (int64_t)batch->batch * tiles * a.groups * 2;
    if (grid > GRID_MAX) return VIPER_INVALID_ARGUMENT;
    const int kv = cache->kv_type;
    const void* fn = cache->head_dim == 64 ? read_fn<64>(kv) : cache->head_dim == 128 ? read_fn<128>(kv) : read_fn<256>(kv);
    void* args[] = {&a};
    launch(fn, (unsigned)grid, KA_NT, 0, (hipStream_t)stream, args);
    return status_of(hipGetLastError());
}
