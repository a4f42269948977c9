// policy.hip — what preference and policy fine-tuning adds to the cross
// entropy: token log-probabilities from logits and their gradient, the
// preference loss of sequence pairs and the clipped policy loss.
#include <math.h>

#include "ta_backend.h"
#include "soft.hpp"
#include "ta_internal.hpp"

namespace ta {

// ── values of a row, 16 bytes at a time ─────────────────────────────────
// Rows start at any multiple of their element (an odd vocabulary), so the
// vectors are declared with the element's alignment: gfx950 loads and stores
// 16 bytes at any address.
template <typename T>
struct Row;
template <>
struct Row<bf16> {
    static constexpr int E = 8;
    typedef uint32_t V4 __attribute__((ext_vector_type(4), aligned(2)));
    static __device__ __forceinline__ void load(const bf16* p, float* f) {
        const V4 v = *(const V4*)p;
#pragma unroll
        for (int i = 0; i < 4; i++) f[2 * i] = lo2f(v[i]), f[2 * i + 1] = hi2f(v[i]);
    }
    static __device__ __forceinline__ void store(bf16* p, const float* f) {
        V4 v;
#pragma unroll
        for (int i = 0; i < 4; i++) v[i] = pack2(f[2 * i], f[2 * i + 1]);
        *(V4*)p = v;
    }
    static __device__ __forceinline__ float one(const bf16* p) { return bf2f(*p); }
    static __device__ __forceinline__ void put(bf16* p, float f) { *p = f2bf(f); }
};
template <>
struct Row<float> {
    static constexpr int E = 4;
    typedef float V4 __attribute__((ext_vector_type(4), aligned(4)));
    static __device__ __forceinline__ void load(const float* p, float* f) {
        const V4 v = *(const V4*)p;
#pragma unroll
        for (int i = 0; i < 4; i++) f[i] = v[i];
    }
    static __device__ __forceinline__ void store(float* p, const float* f) {
        *(V4*)p = (V4){f[0], f[1], f[2], f[3]};
    }
    static __device__ __forceinline__ float one(const float* p) { return *p; }
    static __device__ __forceinline__ void put(float* p, float f) { *p = f; }
};

// statistics of one row over a block of NW waves
template <typename T, int NW, bool ENT>
__device__ __forceinline__ Soft row_soft(const T* L, int V, float c2, Soft* red) {
    constexpr int E = Row<T>::E;
    Soft st = {-INFINITY, 0.f, 0.f};
    const int nv = V / E;
    for (int k = threadIdx.x; k < nv; k += 64 * NW) {
        float f[E];
        Row<T>::load(L + (int64_t)k * E, f);
        soft_add<E, ENT>(st, f, c2);
    }
    for (int i = nv * E + threadIdx.x; i < V; i += 64 * NW) {
        const float f = Row<T>::one(L + i);
        soft_add<1, ENT>(st, &f, c2);
    }
    return soft_block<NW>(st, c2, red);
}

template <typename T, bool ENT>
__global__ __launch_bounds__(512) void k_token_logp(const T* __restrict__ logits, int64_t ld,
                                                    const int32_t* __restrict__ targets, float c,
                                                    float* __restrict__ logp,
                                                    float* __restrict__ lse,
                                                    float* __restrict__ entropy, int N, int V) {
    __shared__ Soft red[8];
    for (int64_t n = blockIdx.x; n < N; n += gridDim.x) {
        const int t = targets[n];
        RowOut o = {0.f, 0.f, 0.f};
        if (t >= 0) {
            const T* L = logits + n * ld;
            const Soft st = row_soft<T, 8, ENT>(L, V, c * kLog2e, red);
            o = row_out(st, t < V ? Row<T>::one(L + t) : 0.f, t < V, c);
        }
        if (threadIdx.x == 0) {
            logp[n] = o.logp;
            lse[n] = o.lse;
            if (ENT) entropy[n] = o.ent;
        }
    }
}

// One row's gradient: c (g [v = t] - p (g + e (log p + H))).
template <typename T>
__device__ __forceinline__ void row_grad(const T* L, T* D, int V, int t, float c, float lse,
                                         float H, float g, float e, int tid, int nt) {
    constexpr int E = Row<T>::E;
    const int nv = V / E;
    for (int k = tid; k < nv; k += nt) {
        float f[E];
        Row<T>::load(L + (int64_t)k * E, f);
#pragma unroll
        for (int q = 0; q < E; q++) {
            const float lp = fmaf(c, f[q], -lse), p = __builtin_amdgcn_exp2f(lp * kLog2e);
            f[q] = c * ((k * E + q == t ? g : 0.f) - p * fmaf(e, fmaxf(lp, kFar) + H, g));
        }
        Row<T>::store(D + (int64_t)k * E, f);
    }
    for (int i = nv * E + tid; i < V; i += nt) {
        const float lp = fmaf(c, Row<T>::one(L + i), -lse);
        const float p = __builtin_amdgcn_exp2f(lp * kLog2e);
        Row<T>::put(D + i, c * ((i == t ? g : 0.f) - p * fmaf(e, fmaxf(lp, kFar) + H, g)));
    }
}
template <typename T>
__device__ __forceinline__ void row_zero(T* D, int V, int tid, int nt) {
    constexpr int E = Row<T>::E;
    float z[E];
#pragma unroll
    for (int q = 0; q < E; q++) z[q] = 0.f;
    const int nv = V / E;
    for (int k = tid; k < nv; k += nt) Row<T>::store(D + (int64_t)k * E, z);
    for (int i = nv * E + tid; i < V; i += nt) Row<T>::put(D + i, 0.f);
}

template <typename T>
__global__ __launch_bounds__(512) void k_token_logp_bwd(
    const T* logits, int64_t ld, const int32_t* __restrict__ targets, float c,
    const float* __restrict__ lse, const float* __restrict__ entropy,
    const float* __restrict__ dlogp, const float* __restrict__ dentropy, T* dlogits, int64_t ldd,
    int N, int V) {
    for (int64_t n = blockIdx.x; n < N; n += gridDim.x) {
        const int t = targets[n];
        float g = 0.f, e = 0.f;
        if (t >= 0) {
            g = dlogp[n];
            if (dentropy) e = dentropy[n];
        }
        T* D = dlogits + n * ldd;
        if (g == 0.f && e == 0.f)
            row_zero(D, V, threadIdx.x, 512);
        else
            row_grad(logits + n * ld, D, V, t, c, lse[n], e != 0.f ? entropy[n] : 0.f, g, e,
                     threadIdx.x, 512);
    }
}

// ── policy loss of one token ────────────────────────────────────────────
struct PolicyArgs {
    const float *old_logp, *ref_logp, *adv, *weight;
    float lo, hi, dual, kl_beta, ent_coef;
};
struct PolicyTok {
    float loss, kl, dlogp;
};
// In 64 bits: exp(d) - d - 1 is a difference of near-equal values at the
// small d of a policy close to its reference.
__device__ __forceinline__ PolicyTok policy_token(const PolicyArgs& a, int64_t n, float logp,
                                                  float ent, float w) {
    const double A = a.adv[n];
    double lr = a.old_logp ? (double)logp - (double)a.old_logp[n] : 0.0;
    const bool far = !(fabs(lr) <= 60.0);
    if (far) lr = lr > 0 ? 60.0 : lr < 0 ? -60.0 : lr;
    const double r = exp(lr), hi = 1.0 + (double)a.hi, lo = 1.0 - (double)a.lo;
    double pg = -fmin(r * A, fmin(fmax(r, lo), hi) * A);
    bool flat = far || (A >= 0 ? r > hi : r < lo);
    if (a.dual > 0.f && A < 0 && r > (double)a.dual) {
        pg = -(double)a.dual * A;
        flat = true;
    }
    // a NaN of the inputs (fmin and the tests drop it) reaches loss and gradient
    double nan = (lr - lr) + (A - A);
    double g = flat ? 0.0 : -A * r, kl = 0.0;
    if (a.ref_logp) {
        double d = (double)a.ref_logp[n] - (double)logp;
        const bool farr = !(fabs(d) <= 60.0);
        if (farr) d = d > 0 ? 60.0 : d < 0 ? -60.0 : d;
        const double em = expm1(d);
        kl = em - d;
        nan += d - d;
        if (!farr) g -= (double)a.kl_beta * em;
    }
    return {(float)(pg + (double)a.kl_beta * kl - (double)a.ent_coef * (double)ent + nan),
            (float)kl, (float)((g + nan) * (double)w)};
}

__global__ __launch_bounds__(256) void k_policy_loss(const float* __restrict__ logp, PolicyArgs a,
                                                     float* __restrict__ loss,
                                                     float* __restrict__ kl,
                                                     float* __restrict__ dlogp, int64_t N) {
    for (int64_t n = blockIdx.x * 256ll + threadIdx.x; n < N; n += gridDim.x * 256ll) {
        const float w = a.weight[n];
        PolicyTok o = {0.f, 0.f, 0.f};
        if (w != 0.f) o = policy_token(a, n, logp[n], 0.f, w);
        if (loss) loss[n] = o.loss;
        if (kl) kl[n] = o.kl;
        dlogp[n] = o.dlogp;
    }
}

template <bool ENT>
__global__ __launch_bounds__(512) void k_policy_logits(const bf16* logits, int64_t ld,
                                                       const int32_t* __restrict__ targets,
                                                       float c, PolicyArgs a,
                                                       float* __restrict__ logp,
                                                       float* __restrict__ entropy,
                                                       float* __restrict__ loss,
                                                       float* __restrict__ kl, bf16* dlogits,
                                                       int64_t ldd, int N, int V) {
    __shared__ Soft red[8];
    __shared__ float sg;
    for (int64_t n = blockIdx.x; n < N; n += gridDim.x) {
        const int t = targets[n];
        const float w = t >= 0 ? a.weight[n] : 0.f;
        const bf16* L = logits + n * ld;
        bf16* D = dlogits + n * ldd;
        RowOut o = {0.f, 0.f, 0.f};
        PolicyTok pt = {0.f, 0.f, 0.f};
        if (w != 0.f) {
            const float ft = t < V ? bf2f(L[t]) : 0.f;
            const Soft st = row_soft<bf16, 8, ENT>(L, V, c * kLog2e, red);
            o = row_out(st, ft, t < V, c);
            if (threadIdx.x == 0) {
                pt = policy_token(a, n, o.logp, ENT ? o.ent : 0.f, w);
                sg = pt.dlogp;
            }
            __syncthreads();
            row_grad(L, D, V, t, c, o.lse, o.ent, sg, ENT ? -a.ent_coef * w : 0.f, threadIdx.x,
                     512);
        } else {
            row_zero(D, V, threadIdx.x, 512);
        }
        if (threadIdx.x == 0) {
            logp[n] = o.logp;
            if (ENT) entropy[n] = o.ent;
            loss[n] = pt.loss;
            if (kl) kl[n] = pt.kl;
        }
        __syncthreads();  // sg is read before the next row writes it
    }
}

// ── preference loss ─────────────────────────────────────────────────────
struct PrefArgs {
    const float *logp, *ref;
    const int32_t* targets;
    const int64_t* offsets;
    int64_t N;
    int kind, average;
    float beta, smoothing, margin, scale;
    float *pair_loss, *rewards, *dlogp;
};
struct PrefSums {
    double pi[2], rf[2];
    int64_t cnt[2];
};
__device__ __forceinline__ double softplus(double z) { return fmax(z, 0.0) + log1p(exp(-fabs(z))); }
// loss and rewards of a pair; du: gradient of scale * loss to pi of the
// chosen answer's sum (or mean), 0 when the pair takes no part
__device__ __forceinline__ double pref_pair(const PrefArgs& a, const PrefSums& q, double* loss,
                                            double* rew) {
    double pi[2], rf[2];
    for (int i = 0; i < 2; i++) {
        const double k = a.average && q.cnt[i] > 0 ? 1.0 / (double)q.cnt[i] : 1.0;
        pi[i] = q.pi[i] * k;
        rf[i] = q.rf[i] * k;
        rew[i] = (double)a.beta * (pi[i] - rf[i]);
    }
    *loss = 0.0;
    if (q.cnt[0] == 0 || q.cnt[1] == 0) return 0.0;
    const double u = (pi[0] - rf[0]) - (pi[1] - rf[1]), beta = a.beta;
    const double z = beta * u - (double)a.margin, sm = a.smoothing;
    double du;
    if (a.kind == TA_PREF_SIGMOID) {
        *loss = (1.0 - sm) * softplus(-z) + sm * softplus(z);
        // sigma(z) - (1 - smoothing), without cancelling at large z
        const double e = exp(-fabs(z)), tail = e / (1.0 + e);
        du = beta * (z >= 0 ? sm - tail : tail - (1.0 - sm));
    } else if (a.kind == TA_PREF_IPO) {
        const double v = u - (double)a.margin - 1.0 / (2.0 * beta);
        *loss = v * v;
        du = 2.0 * v;
    } else {
        *loss = z < 1.0 ? 1.0 - z : z - z;  // (NaN stays)
        du = z < 1.0 ? -beta : z - z;
    }
    return du * (double)a.scale;
}
__device__ __forceinline__ void pref_range(const PrefArgs& a, int64_t q, int64_t* b, int64_t* e) {
    *b = min(max(a.offsets[q], (int64_t)0), a.N);
    *e = min(max(a.offsets[q + 1], *b), a.N);
}
__device__ __forceinline__ int64_t wave_sum_l(int64_t v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
    return v;
}

// One block per pair: sums, loss, gradient.
__global__ __launch_bounds__(256) void k_preference(PrefArgs a) {
    __shared__ double sp[4], sr[4];
    __shared__ int64_t sc[4];
    __shared__ double sdu;
    const int64_t p = blockIdx.x;
    PrefSums q;
    int64_t b[2], e[2];
    for (int i = 0; i < 2; i++) {
        pref_range(a, 2 * p + i, &b[i], &e[i]);
        double pi = 0.0, rf = 0.0;
        int64_t cnt = 0;
        for (int64_t j = b[i] + threadIdx.x; j < e[i]; j += 256)
            if (a.targets[j] >= 0) {
                pi += (double)a.logp[j];
                if (a.ref) rf += (double)a.ref[j];
                cnt++;
            }
        pi = wave_sum_d(pi);
        rf = wave_sum_d(rf);
        cnt = wave_sum_l(cnt);
        __syncthreads();
        if ((threadIdx.x & 63) == 0) {
            sp[threadIdx.x >> 6] = pi;
            sr[threadIdx.x >> 6] = rf;
            sc[threadIdx.x >> 6] = cnt;
        }
        __syncthreads();
        q.pi[i] = ((sp[0] + sp[1]) + sp[2]) + sp[3];
        q.rf[i] = ((sr[0] + sr[1]) + sr[2]) + sr[3];
        q.cnt[i] = sc[0] + sc[1] + sc[2] + sc[3];
    }
    if (threadIdx.x == 0) {
        double loss, rew[2];
        sdu = pref_pair(a, q, &loss, rew);
        a.pair_loss[p] = (float)loss;
        if (a.rewards) {
            a.rewards[2 * p] = (float)rew[0];
            a.rewards[2 * p + 1] = (float)rew[1];
        }
    }
    __syncthreads();
    if (!a.dlogp) return;
    for (int i = 0; i < 2; i++) {
        const double k = a.average && q.cnt[i] > 0 ? 1.0 / (double)q.cnt[i] : 1.0;
        const float g = (float)((i ? -sdu : sdu) * k);
        for (int64_t j = b[i] + threadIdx.x; j < e[i]; j += 256)
            a.dlogp[j] = a.targets[j] >= 0 ? g : 0.f;
    }
}

// at most this many blocks of a launch over rows (its threads stay below 2^32)
static inline dim3 row_grid(int64_t rows) { return dim3((unsigned)(rows < (1 << 20) ? rows : 1 << 20)); }
static bool temp_ok(float c) { return c > 0.f && c < INFINITY; }

template <typename T>
static int token_logp_fwd(const T* logits, int64_t ld, const int32_t* targets, float c, float* logp,
                          float* lse, float* entropy, int N, int V, hipStream_t s) {
    TA_REQUIRE(N >= 0 && V > 0 && ld >= V, "token_logp_fwd: bad shape N=%d V=%d ld=%lld", N, V,
               (long long)ld);
    TA_REQUIRE(temp_ok(c), "token_logp_fwd: inv_temp must be positive and finite");
    if (N == 0) return 0;
    TA_REQUIRE(logits && targets && logp && lse, "token_logp_fwd: null argument");
    TA_REQUIRE(((uintptr_t)logits % sizeof(T)) == 0, "token_logp_fwd: misaligned logits");
    if (entropy)
        tlaunch(k_token_logp<T, true>, row_grid(N), dim3(512), s, logits, ld, targets, c, logp, lse,
                entropy, N, V);
    else
        tlaunch(k_token_logp<T, false>, row_grid(N), dim3(512), s, logits, ld, targets, c, logp,
                lse, entropy, N, V);
    return check_launch("token_logp_fwd");
}

template <typename T>
static int token_logp_bwd(const T* logits, int64_t ld, const int32_t* targets, float c,
                          const float* lse, const float* entropy, const float* dlogp,
                          const float* dentropy, T* dlogits, int64_t ldd, int N, int V,
                          hipStream_t s) {
    TA_REQUIRE(N >= 0 && V > 0 && ld >= V && ldd >= V,
               "token_logp_bwd: bad shape N=%d V=%d ld=%lld ldd=%lld", N, V, (long long)ld,
               (long long)ldd);
    TA_REQUIRE(temp_ok(c), "token_logp_bwd: inv_temp must be positive and finite");
    if (N == 0) return 0;
    TA_REQUIRE(logits && targets && lse && dlogp && dlogits, "token_logp_bwd: null argument");
    TA_REQUIRE(!dentropy || entropy, "token_logp_bwd: dentropy needs the entropy");
    TA_REQUIRE((((uintptr_t)logits | (uintptr_t)dlogits) % sizeof(T)) == 0,
               "token_logp_bwd: misaligned rows");
    TA_REQUIRE(dlogits != logits || ldd == ld, "token_logp_bwd: in place needs ldd = ld");
    tlaunch(k_token_logp_bwd<T>, row_grid(N), dim3(512), s, logits, ld, targets, c, lse, entropy,
            dlogp, dentropy, dlogits, ldd, N, V);
    return check_launch("token_logp_bwd");
}

static int policy_args(const char* what, const float* adv, const float* weight, float lo, float hi,
                       float dual, float kl_beta, float ent_coef) {
    TA_REQUIRE(adv && weight, "%s: null argument", what);
    TA_REQUIRE(lo >= 0.f && lo < 1.f && hi >= 0.f && hi < INFINITY,
               "%s: clip range 1 - %g .. 1 + %g", what, lo, hi);
    TA_REQUIRE(dual == 0.f || (dual > 1.f && dual < INFINITY),
               "%s: dual_clip must be 0 or above 1", what);
    TA_REQUIRE(fabsf(kl_beta) < INFINITY && fabsf(ent_coef) < INFINITY,
               "%s: coefficients must be finite", what);
    return 0;
}

}  // namespace ta

using namespace ta;

extern "C" {

int ta_token_logp_fwd(const uint16_t* logits, int64_t ld, const int32_t* targets, float inv_temp,
                      float* logp, float* lse, float* entropy, int N, int V, void* stream) {
    return token_logp_fwd(logits, ld, targets, inv_temp, logp, lse, entropy, N, V,
                          (hipStream_t)stream);
}
int ta_token_logp_fwd_f32(const float* logits, int64_t ld, const int32_t* targets, float inv_temp,
                          float* logp, float* lse, float* entropy, int N, int V, void* stream) {
    return token_logp_fwd(logits, ld, targets, inv_temp, logp, lse, entropy, N, V,
                          (hipStream_t)stream);
}
int ta_token_logp_bwd(const uint16_t* logits, int64_t ld, const int32_t* targets, float inv_temp,
                      const float* lse, const float* entropy, const float* dlogp,
                      const float* dentropy, uint16_t* dlogits, int64_t ldd, int N, int V,
                      void* stream) {
    return token_logp_bwd(logits, ld, targets, inv_temp, lse, entropy, dlogp, dentropy, dlogits,
                          ldd, N, V, (hipStream_t)stream);
}
int ta_token_logp_bwd_f32(const float* logits, int64_t ld, const int32_t* targets, float inv_temp,
                          const float* lse, const float* entropy, const float* dlogp,
                          const float* dentropy, float* dlogits, int64_t ldd, int N, int V,
                          void* stream) {
    return token_logp_bwd(logits, ld, targets, inv_temp, lse, entropy, dlogp, dentropy, dlogits,
                          ldd, N, V, (hipStream_t)stream);
}

int ta_preference_loss(const float* logp, const float* ref_logp, const int32_t* targets,
                       const int64_t* offsets, int P, int64_t N, int kind, int average, float beta,
                       float smoothing, float margin, float scale, float* pair_loss,
                       float* rewards, float* dlogp, void* stream) {
    TA_REQUIRE(P >= 0 && P <= (1 << 23) && N >= 0, "preference_loss: bad shape P=%d N=%lld", P,
               (long long)N);
    TA_REQUIRE(kind >= TA_PREF_SIGMOID && kind <= TA_PREF_HINGE, "preference_loss: bad kind %d",
               kind);
    TA_REQUIRE(average == 0 || average == 1, "preference_loss: average must be 0 or 1");
    TA_REQUIRE(beta > 0.f && beta < INFINITY, "preference_loss: beta must be positive and finite");
    TA_REQUIRE(smoothing >= 0.f && smoothing < 1.f, "preference_loss: smoothing outside [0, 1)");
    TA_REQUIRE(smoothing == 0.f || kind == TA_PREF_SIGMOID,
               "preference_loss: smoothing is for the sigmoid loss");
    TA_REQUIRE(fabsf(margin) < INFINITY && fabsf(scale) < INFINITY,
               "preference_loss: margin and scale must be finite");
    if (P == 0) return 0;
    TA_REQUIRE(offsets && pair_loss && (N == 0 || (logp && targets)),
               "preference_loss: null argument");
    const PrefArgs a{logp,      ref_logp, targets, offsets, N,         kind,    average, beta,
                     smoothing, margin,   scale,   pair_loss, rewards, dlogp};
    tlaunch(k_preference, dim3(P), dim3(256), (hipStream_t)stream, a);
    return check_launch("preference_loss");
}

int ta_policy_loss(const float* logp, const float* old_logp, const float* ref_logp,
                   const float* adv, const float* weight, float clip_lo, float clip_hi,
                   float dual_clip, float kl_beta, float* loss, float* kl, float* dlogp,
                   int64_t N, void* stream) {
    TA_REQUIRE(N >= 0, "policy_loss: bad shape N=%lld", (long long)N);
    if (N == 0) return 0;
    TA_REQUIRE(logp && dlogp, "policy_loss: null argument");
    if (int rc = policy_args("policy_loss", adv, weight, clip_lo, clip_hi, dual_clip, kl_beta, 0.f))
        return rc;
    const PolicyArgs a{old_logp, ref_logp, adv, weight, clip_lo, clip_hi, dual_clip, kl_beta, 0.f};
    const int64_t blocks = (N + 255) / 256;
    tlaunch(k_policy_loss, row_grid(blocks), dim3(256), (hipStream_t)stream, logp, a, loss, kl,
            dlogp, N);
    return check_launch("policy_loss");
}

int ta_policy_loss_logits(const uint16_t* logits, int64_t ld, const int32_t* targets,
                          float inv_temp, const float* old_logp, const float* ref_logp,
                          const float* adv, const float* weight, float clip_lo, float clip_hi,
                          float dual_clip, float kl_beta, float ent_coef, float* logp,
                          float* entropy, float* loss, float* kl, uint16_t* dlogits, int64_t ldd,
                          int N, int V, void* stream) {
    TA_REQUIRE(N >= 0 && V > 0 && ld >= V && ldd >= V,
               "policy_loss_logits: bad shape N=%d V=%d ld=%lld ldd=%lld", N, V, (long long)ld,
               (long long)ldd);
    TA_REQUIRE(temp_ok(inv_temp), "policy_loss_logits: inv_temp must be positive and finite");
    if (N == 0) return 0;
    TA_REQUIRE(logits && targets && logp && loss && dlogits, "policy_loss_logits: null argument");
    if (int rc = policy_args("policy_loss_logits", adv, weight, clip_lo, clip_hi, dual_clip,
                             kl_beta, ent_coef))
        return rc;
    TA_REQUIRE(ent_coef == 0.f || entropy, "policy_loss_logits: ent_coef needs the entropy");
    TA_REQUIRE((((uintptr_t)logits | (uintptr_t)dlogits) & 1) == 0,
               "policy_loss_logits: misaligned rows");
    TA_REQUIRE(dlogits != logits || ldd == ld, "policy_loss_logits: in place needs ldd = ld");
    const PolicyArgs a{old_logp, ref_logp, adv,       weight,  clip_lo,
                       clip_hi,  dual_clip, kl_beta, ent_coef};
    hipStream_t s = (hipStream_t)stream;
    if (entropy)
        tlaunch(k_policy_logits<true>, row_grid(N), dim3(512), s, logits, ld, targets, inv_temp, a,
                logp, entropy, loss, kl, dlogits, ldd, N, V);
    else
        tlaunch(k_policy_logits<false>, row_grid(N), dim3(512), s, logits, ld, targets, inv_temp, a,
                logp, entropy, loss, kl, dlogits, ldd, N, V);
    return check_launch("policy_loss_logits");
}

}  // extern "C"
