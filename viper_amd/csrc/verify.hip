// Verification of drafted tokens against the target's probabilities, from given
// uniforms (speculative sampling): accept token d_i while u_i q_i(d_i) < p_i(d_i),
// then draw the next token from max(p - q, 0) (or p after the last).
//
// Measured: 8 sequences of up to 15 drafted tokens, 166144 logits, the drafter's logits
// too: 49 us (statistics 21-27, selection 23); one certain draft of 4 tokens, 32000 logits:
// 17 us (4 and 12.5, the latency of the selection's steps; the tokens of an octet
// one after the other, which is half the code, 19.9: their exponentials overlap).
//
// Which token comes out depends on comparisons with cumulated sums over the whole
// vocabulary, so that a sum held in 32 bits would decide some of them by its
// rounding (166144 terms: a few per cent of the draws of a flat row).  Weights e^((l - M) / T)
// and their sums are 64-bit.
//
// Two launches.  verify_stats_kernel: per row and chunk of 4096 logits the
// largest value M_c, its first index and sum_c = sum e^((l - M_c) / T).
// verify_select_kernel, a workgroup per sequence and chunk: every workgroup joins
// the chunks of the sequence's rows (M, Z = sum_c sum_c e^((M_c - M) / T)) and finds
// how many tokens are accepted.  Where the deciding row's weights are p itself
// (nothing rejected, or a certain drafter: p without its token) the sums of its
// chunks are known and the first workgroup goes on alone; else each sums
// max(p - q, 0) over its chunk and the one that counts last goes on: it finds the chunk
// and the token where the cumulated weight passes u times the total, in index order.

#include "qlinear_host.h"

namespace vq {

constexpr int VF_CHUNK = 4096;  // the smaller of the two chunk sizes
constexpr int VF_NT = 256;      // threads of verify_stats_kernel
constexpr int vs_threads(int chunk) { return chunk / 8; }  // of verify_select_kernel
constexpr int VF_CNT = 4096;  // sequences of a call, a counter each

struct VfStat {
    double sum;
    float max;
    int arg;
};

struct VerifyArgs {
    const uint16_t* target;
    const uint16_t* draft;
    const int32_t* tokens;
    const int32_t* lens;
    const float* uniforms;
    const float* temperature;
    int32_t* out;
    int32_t* accepted;
    float* ratios;
    unsigned* cnt;
    VfStat* stats;  // [B][2R - 1][chunks]: the target's rows, then the drafter's
    double* sums;   // [B][chunks]
    int B, R, V, chunks;
};

// Sequence b's temperature and drafted tokens; false where they do not fit
__device__ __forceinline__ bool vf_seq(const VerifyArgs& a, int b, float& T, int& n) {
    T = a.temperature != nullptr ? a.temperature[b] : 1.0f;
    n = a.lens != nullptr ? a.lens[b] : a.R - 1;
    return T >= 0.0f && T < __builtin_inff() && n >= 0 && n < a.R;
}

// N logits from index j of a row, octets `step` octets apart; past the row NaN,
// which weighs nothing
template <bool VEC, int N>
__device__ __forceinline__ void vf_load(const uint16_t* row, int j, int step, int V, float* l) {
    u32x4 v[N / 8];
#pragma unroll
    for (int h = 0; h < N / 8; ++h) {
        const int x = j + 8 * step * h;
        v[h] = u32x4{0xffffffffu, 0xffffffffu, 0xffffffffu, 0xffffffffu};
        if constexpr (VEC) {  // rows of whole octets, 16-byte aligned
            if (x < V) v[h] = *(const u32x4*)(row + x);
        } else {
            uint32_t w[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) w[i] = x + i < V ? row[x + i] : 0xffffu;
            v[h] = u32x4{w[0] | w[1] << 16, w[2] | w[3] << 16, w[4] | w[5] << 16, w[6] | w[7] << 16};
        }
    }
#pragma unroll
    for (int h = 0; h < N / 8; ++h) {
        const uint32_t w[4] = {v[h].x, v[h].y, v[h].z, v[h].w};
#pragma unroll
        for (int i = 0; i < 8; ++i) l[8 * h + i] = bf16f((w[i >> 1] >> (16 * (i & 1))) & 0xffffu);
    }
}

// e^((l - M) / T): 1 at the maximum (also an infinite one), 0 for NaN, for what is
// infinitely far below the maximum at any T, and below 2^-1000.  With y = 64 (l - M)
// log2 e / T = 64 n + k + f, |f| <= 1/2, it is 2^n 2^(k/64) times the power series of
// 2^(f/64) to its 4th term (what is left out is under (ln 2 / 128)^5 / 5! = 4e-14 of
// the weight, so that a token can differ from one drawn by exact weights where the
// uniform lies that close to a border).  What bounds the statistics is the
// number of instructions a logit takes (full drafts of 8 sequences, 21 million
// logits): 64-bit adds and products run at the full rate, conversions, rounding and
// ldexp at a quarter of it.  So l is widened by its bits: placed in a double they
// read as 2^-896 l, exactly, below the normal range too (an infinite l as 2^128, which
// vf_floor takes care of), and 2^896 goes into the factor; the whole part of y is the
// low word of y + 1.5 * 2^52, n goes into the exponent and 2^(k/64) comes from a table
// in LDS.
__device__ const double VF_POW2[64] = {
    1, 1.0108892860517005, 1.0218971486541166, 1.0330248790212284,
    1.0442737824274138, 1.0556451783605572, 1.0671404006768237, 1.0787607977571199,
    1.0905077326652577, 1.1023825833078409, 1.1143867425958924, 1.1265216186082418,
    1.1387886347566916, 1.1511892299529827, 1.1637248587775775, 1.1763969916502812,
    1.189207115002721, 1.2021567314527031, 1.215247359980469, 1.22848053610687,
    1.241857812073484, 1.2553807570246911, 1.2690509571917332, 1.2828700160787783,
    1.2968395546510096, 1.3109612115247644, 1.3252366431597413, 1.3396675240533029,
    1.3542555469368927, 1.3690024229745905, 1.383909881963832, 1.3989796725383112,
    1.4142135623730951, 1.42961333839197, 1.4451808069770467, 1.460917794180647,
    1.4768261459394993, 1.4929077282912648, 1.5091644275934228, 1.5255981507445384,
    1.5422108254079407, 1.5590044002378369, 1.5759808451078865, 1.593142151342267,
    1.6104903319492543, 1.6280274218573478, 1.6457554781539649, 1.6636765803267364,
    1.681792830507429, 1.7001063537185235, 1.7186192981224779, 1.7373338352737062,
    1.7562521603732995, 1.7753764925265212, 1.7947090750031072, 1.8142521755003989,
    1.8340080864093424, 1.8539791250833855, 1.8741676341103, 1.8945759815869656,
    1.9152065613971474, 1.9360617934922943, 1.9571441241754002, 1.9784560263879509};
__device__ __forceinline__ double widen(float l) {
    const uint32_t u = __float_as_uint(l), hi = (u & 0x80000000u) | ((u & 0x7fffffffu) >> 3);
    return __longlong_as_double((long long)((unsigned long long)hi << 32));
}
// 2^896 64 log2 e / T.  It fits in 64 bits down to T = 2^-121; below 2^-120 (what
// only logits under 10^-34 tell apart) that is taken.
__device__ __forceinline__ double vf_c(float T) {
    constexpr double SCALE = 0x1p896 * 64 * 1.4426950408889634074;
    return T > 0.0f ? SCALE / fmax((double)T, 0x1p-120) : 0.0;
}
// The y above which a logit weighs: 2^-1000, or at temperatures where that lies
// further down, what separates -inf from the finite ones, and these from +inf
// (the logits next to an infinite one are 2^120 from it: 64 log2 e 2^120 / T passes
// 64000 up to T = 1.9e33, so that an ordinary temperature waits for no M here)
__device__ __forceinline__ double vf_floor(float M, float T, double c) {
    if (T < 1e33f) return -64000.0;
    const double inf = widen(__builtin_inff());
    const double gap = M == __builtin_inff() ? 0x1p-776 : inf + widen(M);  // (2^120 is the step below 2^128)
    return fmax(-64000.0, -gap * c);
}
// A value that all lanes have, in scalar registers
__device__ __forceinline__ double wave_uniform(double v) {
    const unsigned long long u = (unsigned long long)__double_as_longlong(v);
    const unsigned lo = (unsigned)__builtin_amdgcn_readfirstlane((int)(unsigned)u);
    const unsigned hi = (unsigned)__builtin_amdgcn_readfirstlane((int)(unsigned)(u >> 32));
    return __longlong_as_double((long long)(lo | (unsigned long long)hi << 32));
}
// c = vf_c(T), lo = vf_floor(M, T, c), pow2 the table in LDS
__device__ __forceinline__ double vf_exp(float l, float M, double c, double lo, const double* pow2) {
    constexpr double MAGIC = 6755399441055744.0;
    const double y = (widen(l) - widen(M)) * c, t = y + MAGIC, f = y - (t - MAGIC);
    const uint32_t n = (uint32_t)(unsigned long long)__double_as_longlong(t);
    double p = 5.7328516886404019e-10;  // (ln2 / 64)^4 / 4!
    p = __builtin_fma(p, f, 2.1173137155464774e-07);
    p = __builtin_fma(p, f, 5.8649049550561693e-05);
    p = __builtin_fma(p, f, 0.010830424696249145);
    p = __builtin_fma(p, f, 1.0) * pow2[n & 63u];
    const double e = __longlong_as_double(__double_as_longlong(p) + (long long)((unsigned long long)(uint32_t)((int)n >> 6) << 52));
    return l <= M && y > lo ? e : 0.0;
}

// What a row's weights need: p(j) = weight(l_j, j)
struct VfRow {
    double iz, c, lo;
    float M;
    int arg;
    bool one;  // all on arg
    __device__ __forceinline__ double weight(float l, int j, const double* pow2) const {
        if (one) return j == arg ? 1.0 : 0.0;
        return vf_exp(l, M, c, lo, pow2) * iz;
    }
};

// Over the wave, every lane gets it: lane swaps within rows of 16, then the row
// swaps (no trip through LDS, as a shuffle takes)
template <int CTRL>
__device__ __forceinline__ double dpp_d(double v) {
    const unsigned long long u = (unsigned long long)__double_as_longlong(v);
    const unsigned long long lo = (unsigned)dpp_i<CTRL>((int)(unsigned)u), hi = (unsigned)dpp_i<CTRL>((int)(unsigned)(u >> 32));
    return __longlong_as_double((long long)(lo | hi << 32));
}
template <class F>
__device__ __forceinline__ unsigned swap_rows(unsigned v, F f) {
    auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    v = f(r[0], r[1]);
    r = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    return f(r[0], r[1]);
}
__device__ __forceinline__ double wave_sum(double v) {
    v += dpp_d<DPP_SWAP1>(v);
    v += dpp_d<DPP_SWAP2>(v);
    v += dpp_d<DPP_HALF_MIRROR>(v);
    v += dpp_d<DPP_MIRROR>(v);
    for (int i = 0; i < 2; ++i) {
        const unsigned long long u = (unsigned long long)__double_as_longlong(v);
        const unsigned a = (unsigned)u, b = (unsigned)(u >> 32);
        const auto lo = i == 0 ? __builtin_amdgcn_permlane16_swap(a, a, false, false) : __builtin_amdgcn_permlane32_swap(a, a, false, false);
        const auto hi = i == 0 ? __builtin_amdgcn_permlane16_swap(b, b, false, false) : __builtin_amdgcn_permlane32_swap(b, b, false, false);
        v = __longlong_as_double((long long)((unsigned long long)lo[0] | (unsigned long long)hi[0] << 32)) +
            __longlong_as_double((long long)((unsigned long long)lo[1] | (unsigned long long)hi[1] << 32));
    }
    return v;
}
__device__ __forceinline__ float wave_max(float v) {
    v = fmaxf(v, dpp_f<DPP_SWAP1>(v));
    v = fmaxf(v, dpp_f<DPP_SWAP2>(v));
    v = fmaxf(v, dpp_f<DPP_HALF_MIRROR>(v));
    v = fmaxf(v, dpp_f<DPP_MIRROR>(v));
    return __uint_as_float(
        swap_rows(__float_as_uint(v), [](unsigned a, unsigned b) { return __float_as_uint(fmaxf(__uint_as_float(a), __uint_as_float(b))); }));
}
__device__ __forceinline__ int wave_min(int v) {
    v = min(v, dpp_i<DPP_SWAP1>(v));
    v = min(v, dpp_i<DPP_SWAP2>(v));
    v = min(v, dpp_i<DPP_HALF_MIRROR>(v));
    v = min(v, dpp_i<DPP_MIRROR>(v));
    return (int)swap_rows((unsigned)v, [](unsigned a, unsigned b) { return (unsigned)min((int)a, (int)b); });
}
// Sum over the workgroup, in a fixed order; red holds a value per wave
template <int NT>
__device__ __forceinline__ double wg_sum(double v, double* red) {
    v = wave_sum(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    double t = red[0];
#pragma unroll
    for (int w = 1; w < NT / 64; ++w) t += red[w];
    return t;
}
// Inclusive sum over the threads before and at this one
__device__ __forceinline__ double wg_scan(double v, double* red) {
    const int lane = (int)threadIdx.x & 63, wave = (int)threadIdx.x >> 6;
    for (int off = 1; off < 64; off <<= 1) {
        const double o = __shfl_up(v, off, 64);
        if (lane >= off) v += o;
    }
    __syncthreads();
    if (lane == 63) red[wave] = v;
    __syncthreads();
    double before = 0.0;
    for (int w = 0; w < wave; ++w) before += red[w];
    return before + v;
}

template <bool VEC, int CH>
__global__ void __launch_bounds__(VF_NT)
verify_stats_kernel(VerifyArgs a) {
    constexpr int PT = CH / VF_NT, W = VF_NT / 64;
    __shared__ float smax[W];
    __shared__ int sarg[W];
    __shared__ double ssum[W], pow2[64];
    const int c = (int)blockIdx.x % a.chunks, rid = (int)blockIdx.x / a.chunks;
    const int per = a.draft != nullptr ? 2 * a.R - 1 : a.R;  // rows of a sequence
    const int b = rid / per, i = rid % per, tid = (int)threadIdx.x, wave = tid >> 6;
    float T;
    int n;
    if (!vf_seq(a, b, T, n)) return;
    if (i < a.R ? i > n : i - a.R >= n) return;
    const uint16_t* row = i < a.R ? a.target + ((size_t)b * a.R + i) * a.V : a.draft + ((size_t)b * (a.R - 1) + i - a.R) * a.V;
    const int j0 = c * CH + tid * 8;
    float l[PT];
    vf_load<VEC, PT>(row, j0, VF_NT, a.V, l);
    if (tid < 64) pow2[tid] = VF_POW2[tid];
    lds_barrier();
    // each wave by its own maximum; the waves meet at the end
    float m = -__builtin_inff();
#pragma unroll
    for (int k = 0; k < PT; ++k) m = fmaxf(m, l[k]);
    m = wave_max(m);
    int arg = 0x7fffffff;
#pragma unroll
    for (int k = PT - 1; k >= 0; --k)
        if (l[k] == m) arg = j0 + (k / 8) * VF_NT * 8 + k % 8;
    arg = wave_min(arg);
    double sum = 0.0;
    if (T > 0.0f && m > -__builtin_inff()) {
        const double e = vf_c(T), lo = wave_uniform(vf_floor(m, T, e));
#pragma unroll
        for (int k = 0; k < PT; ++k) sum += vf_exp(l[k], m, e, lo, pow2);
        sum = wave_sum(sum);
    }
    if ((tid & 63) == 0) {
        smax[wave] = m;
        sarg[wave] = arg;
        ssum[wave] = sum;
    }
    __syncthreads();
    if (tid == 0) {
        const double e = vf_c(T);
        float M = smax[0];
        for (int w = 1; w < W; ++w) M = fmaxf(M, smax[w]);
        const double lo = vf_floor(M, T, e);
        double z = 0.0;
        arg = 0x7fffffff;
        for (int w = 0; w < W; ++w) {
            z += ssum[w] * vf_exp(smax[w], M, e, lo, pow2);
            if (smax[w] == M) arg = min(arg, sarg[w]);
        }
        a.stats[((size_t)b * (2 * a.R - 1) + i) * a.chunks + c] = VfStat{z, M, arg};
    }
}

template <bool VEC, int CH>
__global__ void __launch_bounds__(vs_threads(CH))
verify_select_kernel(VerifyArgs a) {
    constexpr int VS_NT = vs_threads(CH), VS_PT = CH / VS_NT;
    constexpr int W = VS_NT / 64, RPW = (2 * VIPER_QLINEAR_MAX_M + W - 1) / W;  // rows of a wave
    __shared__ VfRow rows[2 * VIPER_QLINEAR_MAX_M];
    __shared__ int taken[VIPER_QLINEAR_MAX_M];
    __shared__ double red[W], pow2[64];
    __shared__ int pick, last_part;
    __shared__ double before;
    const int c = (int)blockIdx.x % a.chunks, b = (int)blockIdx.x / a.chunks;
    const int tid = (int)threadIdx.x, lane = tid & 63, wave = tid >> 6;
    int32_t* out = a.out + (size_t)b * a.R;
    float T;
    int n;
    if (!vf_seq(a, b, T, n)) {
        if (c == 0) {
            if (tid < a.R) out[tid] = -1;
            if (tid == 0) a.accepted[b] = -1;
            if (a.ratios != nullptr && tid < a.R - 1) a.ratios[(size_t)b * (a.R - 1) + tid] = 0.0f;
        }
        return;
    }
    const double e = vf_c(T);
    if (tid < 64) pow2[tid] = VF_POW2[tid];
    lds_barrier();
    const VfStat* stats = a.stats + (size_t)b * (2 * a.R - 1) * a.chunks;
    const uint16_t* trow = a.target + (size_t)b * a.R * a.V;
    const uint16_t* drow = a.draft != nullptr ? a.draft + (size_t)b * (a.R - 1) * a.V : nullptr;
    int dtoken = -1;
    float dp = 0.0f, dq = 0.0f, du = 0.0f;
    if (tid < n) {  // (in flight while the rows are joined)
        dtoken = a.tokens[(size_t)b * (a.R - 1) + tid];
        du = a.uniforms[(size_t)b * a.R + tid];
        if (dtoken >= 0 && dtoken < a.V) {
            dp = bf16f(trow[(size_t)tid * a.V + dtoken]);
            if (drow != nullptr) dq = bf16f(drow[(size_t)tid * a.V + dtoken]);
        }
    }

    // the rows' maxima and sums: rows 0 .. n of the target, n of the drafter; a wave
    // has up to RPW rows, a lane every 64th chunk, the first of which is loaded
    // for all of them at once
    const int nrows = n + 1 + (drow != nullptr ? n : 0);
    auto row_stats = [&](int k) { return stats + (size_t)(k <= n ? k : a.R + k - n - 1) * a.chunks; };
    VfStat head[RPW];
#pragma unroll
    for (int i = 0; i < RPW; ++i) {
        const int k = wave + i * W;
        head[i] = VfStat{0.0, -__builtin_inff(), 0x7fffffff};
        if (k < nrows && lane < a.chunks) head[i] = row_stats(k)[lane];
    }
#pragma unroll
    for (int i = 0; i < RPW; ++i) {
        const int k = wave + i * W;
        if (k >= nrows) break;
        const VfStat* s = row_stats(k);
        float M = head[i].max;
        int arg = head[i].max > -__builtin_inff() ? head[i].arg : 0x7fffffff;
        for (int x = lane + 64; x < a.chunks; x += 64) {
            const VfStat v = s[x];
            if (v.max > M) {  // (chunks in index order: the first of equal ones stays)
                M = v.max;
                arg = v.arg;
            }
        }
        const float mine = M;
        M = wave_max(M);
        arg = wave_min(mine == M ? arg : 0x7fffffff);
        const double lo = vf_floor(M, T, e);
        double z = head[i].sum * vf_exp(head[i].max, M, e, lo, pow2);
        for (int x = lane + 64; x < a.chunks; x += 64) z += s[x].sum * vf_exp(s[x].max, M, e, lo, pow2);
        z = wave_sum(z);
        if (lane == 0) {
            VfRow r;
            r.M = M;
            r.c = e;
            r.lo = lo;
            r.iz = 1.0 / z;
            const bool none = !(M > -__builtin_inff());
            r.arg = none ? 0 : arg;
            r.one = none || T == 0.0f;
            rows[k] = r;
        }
    }
    __syncthreads();
    if (tid < n) {
        double p = 0.0, q = 1.0;
        if (dtoken >= 0 && dtoken < a.V) {
            p = rows[tid].weight(dp, dtoken, pow2);
            if (drow != nullptr) q = rows[n + 1 + tid].weight(dq, dtoken, pow2);
        }
        taken[tid] = (double)du * q < p;
        if (c == 0 && a.ratios != nullptr)
            a.ratios[(size_t)b * (a.R - 1) + tid] = p > 0.0 ? (float)fmin(1.0, p / q) : 0.0f;
    } else if (c == 0 && a.ratios != nullptr && tid < a.R - 1) {
        a.ratios[(size_t)b * (a.R - 1) + tid] = 0.0f;
    }
    __syncthreads();
    int r = 0;  // the deciding row
    while (r < n && taken[r]) ++r;
    VfRow pr = rows[r];
    pr.lo = wave_uniform(pr.lo);
    const bool less = r < n;  // a rejected token: what the drafter gave is taken away
    const bool point = less && drow == nullptr;
    const bool alone = !less || point;
    if (alone && c != 0) return;
    const int dtok = less ? a.tokens[(size_t)b * (a.R - 1) + r] : -1;
    VfRow qr = pr;
    if (less && drow != nullptr) {
        qr = rows[n + 1 + r];
        qr.lo = wave_uniform(qr.lo);
    }
    const uint16_t* prow = trow + (size_t)r * a.V;
    const uint16_t* qrow = less && drow != nullptr ? drow + (size_t)r * a.V : nullptr;

    // weights of consecutive tokens; plain: the target's own
    auto weights = [&](int j, bool plain, double* w) {
        float l[VS_PT], ld[VS_PT];
        vf_load<VEC, VS_PT>(prow, j, 1, a.V, l);
        if (!plain && qrow != nullptr) vf_load<VEC, VS_PT>(qrow, j, 1, a.V, ld);
#pragma unroll
        for (int k = 0; k < VS_PT; ++k) {
            double v = j + k < a.V ? pr.weight(l[k], j + k, pow2) : 0.0;
            if (!plain && less && j + k < a.V) {
                const double q = point ? (j + k == dtok ? 1.0 : 0.0) : qr.weight(ld[k], j + k, pow2);
                v = fmax(v - q, 0.0);
            }
            w[k] = v;
        }
    };
    double w[VS_PT], sum = 0.0;
    double* sums = a.sums + (size_t)b * a.chunks;
    double without = 0.0;  // the sum of the rejected token's chunk without it
    const int dchunk = point && dtok >= 0 && dtok < a.V ? dtok / CH : -1;
    if (!alone || dchunk >= 0) {
        weights((alone ? dchunk : c) * CH + tid * VS_PT, false, w);
#pragma unroll
        for (int k = 0; k < VS_PT; ++k) sum += w[k];
        without = wg_sum<VS_NT>(sum, red);
    }
    if (!alone) {
        // written through to where every XCD sees it, and counted once it is there
        if (tid == 0) {
            __hip_atomic_store((unsigned long long*)sums + c, (unsigned long long)__double_as_longlong(without), __ATOMIC_RELAXED,
                               __HIP_MEMORY_SCOPE_AGENT);
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            const unsigned old = __hip_atomic_fetch_add(a.cnt + b, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            last_part = old == (unsigned)(a.chunks - 1);
            if (last_part) __hip_atomic_store(a.cnt + b, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        }
        __syncthreads();
        if (!last_part) return;
    }

    // the chunk: threads hold consecutive runs of chunk sums
    const int run = (a.chunks + VS_NT - 1) / VS_NT, x0 = min(tid * run, a.chunks), x1 = min(x0 + run, a.chunks);
    bool plain = false;
    double mine = 0.0, scan = 0.0, total = 0.0;
    auto chunk_sum = [&](int x) {
        if (!plain && !alone)
            return __longlong_as_double((long long)__hip_atomic_load((unsigned long long*)sums + x, __ATOMIC_RELAXED,
                                                                     __HIP_MEMORY_SCOPE_AGENT));
        if (!plain && x == dchunk) return without;
        const VfStat v = stats[(size_t)r * a.chunks + x];
        if (pr.one) return pr.arg / CH == x ? 1.0 : 0.0;
        return v.sum * vf_exp(v.max, pr.M, e, pr.lo, pow2) * pr.iz;
    };
    for (int pass = 0; pass < 2; ++pass) {
        mine = 0.0;
        for (int x = x0; x < x1; ++x) mine += chunk_sum(x);
        scan = wg_scan(mine, red);
        __syncthreads();
        if (tid == VS_NT - 1) before = scan;
        __syncthreads();
        total = before;
        if (total > 0.0) break;
        plain = true;  // nothing left of the target's weights: the target's own
    }
    const double u = fmax(0.0, (double)a.uniforms[(size_t)b * a.R + a.R - 1]);
    double goal = u * total;
    if (tid == 0) pick = 0x7fffffff;
    __syncthreads();
    if (mine > 0.0 && scan > goal) atomicMin(&pick, tid);
    __syncthreads();
    if (pick != 0x7fffffff) {
        if (tid == pick) {
            // the chunk within this thread's run: its sums are added up again from
            // what comes before them
            double acc = scan - mine;
            for (int x = x0; x < x1; ++x) {
                const double v = chunk_sum(x);
                if (!(v > 0.0)) continue;
                before = acc;
                last_part = x;
                acc += v;
                if (acc > goal) break;
            }
        }
    } else {  // u * total rounded up to the total: the last chunk with a weight
        __syncthreads();
        if (tid == 0) pick = -1;
        __syncthreads();
        int lastx = -1;
        for (int x = x0; x < x1; ++x)
            if (chunk_sum(x) > 0.0) lastx = x;
        if (lastx >= 0) atomicMax(&pick, lastx);
        __syncthreads();
        if (tid == 0) {
            last_part = pick < 0 ? 0 : pick;
            before = 0.0;
        }
        goal = __builtin_inf();
    }
    __syncthreads();
    const int ch = last_part;
    const double base = before;
    const int j0 = ch * CH + tid * VS_PT;
    weights(j0, plain, w);
    sum = 0.0;
    int mylast = -1;
#pragma unroll
    for (int k = 0; k < VS_PT; ++k) {
        sum += w[k];
        if (w[k] > 0.0) mylast = j0 + k;
    }
    scan = base + wg_scan(sum, red);
    __syncthreads();
    if (tid == 0) pick = 0x7fffffff;
    __syncthreads();
    if (mylast >= 0 && scan > goal) {
        // the first token of this thread that passes; its last one where the
        // additions' order hides it
        double acc = scan - sum;
        int j = mylast;
#pragma unroll
        for (int k = 0; k < VS_PT; ++k) {
            acc += w[k];
            if (w[k] > 0.0 && acc > goal && j0 + k < j) j = j0 + k;
        }
        atomicMin(&pick, j);
    }
    __syncthreads();
    if (pick == 0x7fffffff) {  // the chunk's last token with a weight
        __syncthreads();
        if (tid == 0) pick = -1;
        __syncthreads();
        if (mylast >= 0) atomicMax(&pick, mylast);
        __syncthreads();
    }
    const int token = pick < 0 ? pr.arg : pick;
    if (tid < a.R) out[tid] = tid < r ? a.tokens[(size_t)b * (a.R - 1) + tid] : tid == r ? token : -1;
    if (tid == 0) a.accepted[b] = r;
}

static int64_t vf_chunks(int V, int chunk = VF_CHUNK) { return ((int64_t)V + chunk - 1) / chunk; }
static bool vf_sizes(int B, int R, int V) {
    return B > 0 && B <= VF_CNT && R > 0 && R <= VIPER_QLINEAR_MAX_M && V > 0 && V < 1 << 26 &&
           (int64_t)B * (2 * R - 1) * vf_chunks(V) <= 1 << 22;  // (launches stay under 2^32 threads)
}
static size_t vf_bytes(int B, int R, int V) {
    const size_t ch = (size_t)vf_chunks(V);
    return VF_CNT * 4 + (size_t)B * (2 * R - 1) * ch * sizeof(VfStat) + (size_t)B * ch * 8;
}

}  // namespace vq

extern "C" size_t viper_hip_verify_workspace_bytes(int B, int R, int V) {
    return vq::vf_sizes(B, R, V) ? vq::vf_bytes(B, R, V) : 0;
}

extern "C" int viper_hip_verify_draft(const void* target_bf16, const void* draft_bf16, const int32_t* draft_tokens,
                                      const int32_t* draft_lens, const float* uniforms, const float* temperature, int B,
                                      int R, int V, int32_t* out_tokens, int32_t* out_accepted, float* accept_probs,
                                      void* workspace, size_t workspace_bytes, void* stream) {
    using namespace vq;
    if (target_bf16 == nullptr || uniforms == nullptr || out_tokens == nullptr || out_accepted == nullptr)
        return VIPER_INVALID_ARGUMENT;
    if (!vf_sizes(B, R, V) || (R > 1 && draft_tokens == nullptr)) return VIPER_INVALID_ARGUMENT;
    if (misaligned(target_bf16, 2) || misaligned(draft_bf16, 2) || misaligned(draft_tokens, 4) || misaligned(draft_lens, 4) ||
        misaligned(uniforms, 4) || misaligned(temperature, 4) || misaligned(out_tokens, 4) || misaligned(out_accepted, 4) ||
        misaligned(accept_probs, 4))
        return VIPER_INVALID_ARGUMENT;
    if (workspace == nullptr || misaligned(workspace, 16) || workspace_bytes < vf_bytes(B, R, V)) return VIPER_INVALID_ARGUMENT;
    // what is written (the first four) overlaps nothing else: other workgroups may still read it
    const size_t rows4 = (size_t)B * R * 4, drafted = (size_t)B * (R - 1);
    const struct {
        const void* p;
        size_t bytes;
    } at[] = {{out_tokens, rows4}, {out_accepted, (size_t)B * 4}, {accept_probs, drafted * 4}, {workspace, vf_bytes(B, R, V)},
              {target_bf16, (size_t)B * R * V * 2}, {draft_bf16, drafted * V * 2}, {draft_tokens, drafted * 4},
              {draft_lens, (size_t)B * 4}, {uniforms, rows4}, {temperature, (size_t)B * 4}};
    for (size_t i = 0; i < 4; ++i)
        for (size_t j = i + 1; j < sizeof(at) / sizeof(at[0]); ++j)
            if (at[i].p != nullptr && at[j].p != nullptr && at[i].bytes != 0 && at[j].bytes != 0 &&
                (uintptr_t)at[i].p < (uintptr_t)at[j].p + at[j].bytes && (uintptr_t)at[j].p < (uintptr_t)at[i].p + at[i].bytes)
                return VIPER_INVALID_ARGUMENT;
    VerifyArgs a;
    a.target = (const uint16_t*)target_bf16;
    a.draft = R > 1 ? (const uint16_t*)draft_bf16 : nullptr;
    a.tokens = draft_tokens;
    a.lens = draft_lens;
    a.uniforms = uniforms;
    a.temperature = temperature;
    a.out = out_tokens;
    a.accepted = out_accepted;
    a.ratios = accept_probs;
    a.B = B;
    a.R = R;
    a.V = V;
    const unsigned rows = (unsigned)B * (R > 1 && draft_bf16 != nullptr ? 2 * R - 1 : R);
    // larger chunks where there are more of them than the GPU holds workgroups
    const bool large = (int64_t)rows * vf_chunks(V) > 8 * device_cus();
    a.chunks = (int)vf_chunks(V, large ? 2 * VF_CHUNK : VF_CHUNK);
    a.cnt = (unsigned*)workspace;
    a.stats = (VfStat*)((char*)workspace + VF_CNT * 4);
    a.sums = (double*)(a.stats + (size_t)B * (2 * R - 1) * a.chunks);
    const bool vec = V % 8 == 0 && !misaligned(target_bf16, 16) && !misaligned(draft_bf16, 16);
    void* args[] = {&a};
    const void* st = large ? (vec ? (const void*)verify_stats_kernel<true, 2 * VF_CHUNK> : (const void*)verify_stats_kernel<false, 2 * VF_CHUNK>)
                           : (vec ? (const void*)verify_stats_kernel<true, VF_CHUNK> : (const void*)verify_stats_kernel<false, VF_CHUNK>);
    const void* se = large ? (vec ? (const void*)verify_select_kernel<true, 2 * VF_CHUNK> : (const void*)verify_select_kernel<false, 2 * VF_CHUNK>)
                           : (vec ? (const void*)verify_select_kernel<true, VF_CHUNK> : (const void*)verify_select_kernel<false, VF_CHUNK>);
    launch(st, rows * (unsigned)a.chunks, VF_NT, 0, (hipStream_t)stream, args);
    const int rc = status_of(hipGetLastError());
    if (rc != VIPER_OK) return rc;
    launch(se, (unsigned)B * (unsigned)a.chunks, vs_threads(large ? 2 * VF_CHUNK : VF_CHUNK), 0, (hipStream_t)stream, args);
    return status_of(hipGetLastError());
}
