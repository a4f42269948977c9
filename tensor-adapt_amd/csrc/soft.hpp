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
// n values f into st; ENT: u too
template <int n, bool ENT>
__device__ __forceinline__ void soft_add(Soft& st, const float* f, float c2) {
    float gm = f[0];
#pragma unroll
    for (int e = 1; e < n; e++) gm = fmaxf(gm, f[e]);
    if (gm > st.m) {
        const float d = st.m - gm, k = __builtin_amdgcn_exp2f(d * c2);
        if (ENT) st.u = k * (st.u + st.s * fmaxf(d, kFar));
        st.s *= k;
        st.m = gm;
    }
    const float R = soft_ref(st.m);
#pragma unroll
    for (int e = 0; e < n; e++) {
        const float d = f[e] - R, p = __builtin_amdgcn_exp2f(d * c2);
        st.s += p;
        if (ENT) st.u = fmaf(p, fmaxf(d, kFar), st.u);
    }
}
template <int NW>
__device__ __forceinline__ Soft soft_block(Soft st, float c2, Soft* red) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        const Soft b = {__shfl_xor(st.m, o, 64), __shfl_xor(st.s, o, 64), __shfl_xor(st.u, o, 64)};
        st = soft_merge(st, b, c2);
    }
    __syncthreads();  // red is free
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = st;
    __syncthreads();
    st = red[0];
#pragma unroll
    for (int k = 1; k < NW; k++) st = soft_merge(st, red[k], c2);
    return st;
}

struct RowOut {
    float logp, lse, ent;
};
__device__ __forceinline__ RowOut row_out(const Soft& st, float ft, bool has_t, float c) {
    const float ls = st.s > 0.f || st.s != st.s ? logf(st.s) : NAN;  // nothing above -Inf
    RowOut o;
    o.logp = has_t ? c * (ft - st.m) - ls : NAN;
    o.lse = c * st.m + ls;
    o.ent = ls - c * (st.u / st.s);
    return o;
}

}  // namespace ta
