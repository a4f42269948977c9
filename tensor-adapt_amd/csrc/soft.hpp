// soft.hpp — softmax statistics of a row of logits, shared by the kernels that
// read logits (policy.hip) and the GEMM that only forms them (gemm.hip).
//
// With x = c f (c = inv_temp) and M = max f of the row:
//   S = sum exp(c (f - M)),  U = sum exp(c (f - M)) (f - M),
//   lse = c M + log S,  logp = c (f_t - M) - log S,  entropy = log S - c U / S.
// The differences are formed before the scaling, so a confident token's logp
// keeps its digits and logits of the type's lowest value do not overflow.
// Partial statistics over any parts of the row merge into the row's.
#pragma once
#include <math.h>

#include "ta_common.hpp"

namespace ta {

// c log2(e) for the eight values of a vector.  Rounded to one F32 the factor is
// off by up to 2^-24, the same way for every logit, and log S by that times the
// mean of |c d|: of the sums' errors the one that does not average out, and a
// policy near its reference shows it in the KL term.  So k of eight values take
// the F32 above it and the others the F32 below, which leaves a sixteenth of
// their distance at most and costs no instruction (a second product with the
// factor's remainder made the forward 6% slower).
struct ExpScale {
    float c[8];
    float near;  // the nearest F32, for single factors
};
inline ExpScale exp_scale(float c) {
    const double x = (double)c * 1.44269504088896340736;
    ExpScale r;
    r.near = (float)fmin(x, 3.4028234663852886e38);
    const float lo = (double)r.near > x ? nextafterf(r.near, 0.f) : r.near;
    const float up = fminf(nextafterf(lo, INFINITY), 3.4028234663852886e38f);
    const int k = up > lo ? (int)lrint(8 * (x - (double)lo) / ((double)up - (double)lo)) : 0;
    // (in the order 0 4 2 6 1 5 3 7, so that the first four are near k / 8 too)
    for (int e = 0; e < 8; e++) {
        const int order = (e & 1) << 2 | (e & 2) | e >> 2;
        r.c[e] = order < k || lo == 0.f ? up : lo;
    }
    return r;  // (none is 0: a logit of -Inf gives exp(-Inf), not 0 * -Inf)
}

// m: maximum (-Inf: none yet), s, u: the sums above relative to m, u without
// the factor c.  c2 = c log2(e): exp(c d) = exp2(c2 d), one v_exp_f32.
struct Soft {
    float m, s, u;
};
constexpr float kFar = -1e30f;  // stands for -Inf where 0 * -Inf would be NaN
__device__ __forceinline__ float soft_ref(float m) { return m == -INFINITY ? 0.f : m; }
__device__ __forceinline__ Soft soft_merge(const Soft& a, const Soft& b, float c2) {
    const float M = fmaxf(a.m, b.m), R = soft_ref(M);
    const float da = a.m - R, db = b.m - R;
    const float fa = __builtin_amdgcn_exp2f(da * c2), fb = __builtin_amdgcn_exp2f(db * c2);
    return {M, a.s * fa + b.s * fb,
            fa * (a.u + a.s * fmaxf(da, kFar)) + fb * (b.u + b.s * fmaxf(db, kFar))};
}
// n values f into st; ENT: u too.  S is joined from the n values' own sum: added
// one by one they would round n times beside what may be nearly all of S.
template <int n, bool ENT>
__device__ __forceinline__ void soft_add(Soft& st, const float* f, const ExpScale& c2) {
    float gm = f[0];
#pragma unroll
    for (int e = 1; e < n; e++) gm = fmaxf(gm, f[e]);
    if (gm > st.m) {
        const float d = st.m - gm, k = __builtin_amdgcn_exp2f(d * c2.near);
        if (ENT) st.u = k * (st.u + st.s * fmaxf(d, kFar));
        st.s *= k;
        st.m = gm;
    }
    const float R = soft_ref(st.m);
    float s = 0.f;
#pragma unroll
    for (int e = 0; e < n; e++) {
        const float d = f[e] - R, p = __builtin_amdgcn_exp2f(d * c2.c[e]);
        s += p;
        if (ENT) st.u = fmaf(p, fmaxf(d, kFar), st.u);
    }
    st.s += s;
}
// Row statistics: S and U in 64 bits, since a sequence adds up the errors of
// its rows' log S and the KL term divides them by small differences.
struct SoftRow {
    float m;
    double s, u;
};
// A block's maximum and sums, for every thread (redm, red: LDS, one entry per
// wave; one barrier each).  NW (a power of two) lanes read the waves' entries
// and a butterfly joins them: every lane reading all of them takes 64
// registers, which a row held in registers spills for.
template <int NW>
__device__ __forceinline__ float block_maxf(float m, float* redm) {
    m = wave_max(m);
    if ((threadIdx.x & 63) == 0) redm[threadIdx.x >> 6] = m;
    __syncthreads();
    m = redm[threadIdx.x & (NW - 1)];
#pragma unroll
    for (int o = NW / 2; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor(m, o, 64));
    return m;
}
template <int NW, bool ENT>
__device__ __forceinline__ SoftRow block_sums(float m, float s1, float u1, double (*red)[2]) {
    const double s = wave_sum_d((double)s1), u = ENT ? wave_sum_d((double)u1) : 0.0;
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6][0] = s, red[threadIdx.x >> 6][1] = u;
    __syncthreads();
    const int k = threadIdx.x & (NW - 1);
    SoftRow r = {m, red[k][0], red[k][1]};
#pragma unroll
    for (int o = NW / 2; o > 0; o >>= 1) {
        r.s += __shfl_xor(r.s, o, 64);
        if (ENT) r.u += __shfl_xor(r.u, o, 64);
    }
    return r;
}
// the statistics of a block's threads merged: the maximum first, then the
// sums (each thread rescales its own once)
template <int NW, bool ENT>
__device__ __forceinline__ SoftRow soft_block(const Soft& st, float c2, float* redm,
                                              double (*red)[2]) {
    const float m = block_maxf<NW>(st.m, redm);
    const float d = st.m - soft_ref(m), f = __builtin_amdgcn_exp2f(d * c2);
    return block_sums<NW, ENT>(m, st.s * f, f * (st.u + st.s * fmaxf(d, kFar)), red);
}

// exp and log in 64 bits to about 1e-11 relative, for the one thread of a
// block that finishes a row: Taylor's series after the usual reduction, a
// handful of registers where the library's take some 60, which rows held in
// registers do not have to spare (the policy kernel spilled 84 to 142 of 128
// registers around them and ran twice as long).
__device__ __forceinline__ double exp_small(double x) {  // |x| <= 0.35
    double p = 1.0 / 3628800.0;
    p = fma(p, x, 1.0 / 362880.0);
    p = fma(p, x, 1.0 / 40320.0);
    p = fma(p, x, 1.0 / 5040.0);
    p = fma(p, x, 1.0 / 720.0);
    p = fma(p, x, 1.0 / 120.0);
    p = fma(p, x, 1.0 / 24.0);
    p = fma(p, x, 1.0 / 6.0);
    p = fma(p, x, 0.5);
    p = fma(p, x, 1.0);
    return fma(p, x, 1.0);
}
constexpr double kLn2 = 0.69314718055994530942;
__device__ __forceinline__ double exp_d(double x) {  // |x| <= 700
    const double n = rint(x * (1.0 / kLn2));
    return ldexp(exp_small(fma(n, -kLn2, x)), (int)n);
}
// From log2 in F32, L: log S = L ln 2 + log(S 2^-L), the last term by its
// series at a value within 2e-6 of 1.
__device__ __forceinline__ double log_d(double S) {
    const float L = __builtin_amdgcn_logf((float)S), n = rintf(L);
    const double e = ldexp(exp_small((double)(n - L) * kLn2), -(int)n);
    const double t = fma(S, e, -1.0);
    return fma((double)L, kLn2, fma(-0.5 * t, t, t));
}

struct RowOut {
    double logp;
    float lse, ent;
};
__device__ __forceinline__ RowOut row_out(const SoftRow& st, float ft, bool has_t, float c) {
    // (nothing above -Inf: NaN)
    const double ls = st.s > 0.0 || st.s != st.s ? log_d(st.s) : (double)NAN;
    RowOut o;
    o.logp = has_t ? (double)c * ((double)ft - (double)st.m) - ls : (double)NAN;
    o.lse = (float)((double)c * (double)st.m + ls);
    o.ent = (float)(ls - (double)(c * ((float)st.u / (float)st.s)));
    return o;
}

}  // namespace ta
