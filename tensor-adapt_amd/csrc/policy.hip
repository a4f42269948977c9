// policy.hip — what preference and policy fine-tuning adds to the cross
// entropy: token log-probabilities from logits and their gradient, the
// preference loss of sequence pairs and the clipped policy loss.
#include <math.h>

#include <algorithm>

#include "ta_backend.h"
#include "soft.hpp"
#include "ta_internal.hpp"

namespace ta {

// Logits are read past the caches (NT: a non-temporal load) where they are
// more than the 256 MB last-level cache holds, so that nothing is kept that the
// next pass will not find: 4096 x 151,936 forward 142 -> 131 us, 2048 x 152,064
// forward and gradient 296 -> 286 us; what fits is faster with plain loads (777
// x 50,257 F32, 156 MB: 67 us against 87).  Gradients are always stored so:
// they are read by a later kernel, and 2048 x 151,936 took 264 us instead of
// 237 with plain stores, 777 x 50,257 F32 83 instead of 67.
constexpr int64_t kCacheBytes = int64_t(256) << 20;

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
    template <bool NT>
    static __device__ __forceinline__ V4 ld(const bf16* p) {
        if constexpr (NT) return __builtin_nontemporal_load((const V4*)p);
        return *(const V4*)p;
    }
    static __device__ __forceinline__ void unpack(const V4& v, float* f) {
#pragma unroll
        for (int i = 0; i < 4; i++) f[2 * i] = lo2f(v[i]), f[2 * i + 1] = hi2f(v[i]);
    }
    static __device__ __forceinline__ void store(bf16* p, const float* f) {
        V4 v;
#pragma unroll
        for (int i = 0; i < 4; i++) v[i] = pack2(f[2 * i], f[2 * i + 1]);
        __builtin_nontemporal_store(v, (V4*)p);
    }
    static __device__ __forceinline__ float one(const bf16* p) { return bf2f(*p); }
    static __device__ __forceinline__ void put(bf16* p, float f) { *p = f2bf(f); }
};
template <>
struct Row<float> {
    static constexpr int E = 4;
    typedef float V4 __attribute__((ext_vector_type(4), aligned(4)));
    template <bool NT>
    static __device__ __forceinline__ V4 ld(const float* p) {
        if constexpr (NT) return __builtin_nontemporal_load((const V4*)p);
        return *(const V4*)p;
    }
    static __device__ __forceinline__ void unpack(const V4& v, float* f) {
#pragma unroll
        for (int i = 0; i < 4; i++) f[i] = v[i];
    }
    static __device__ __forceinline__ void store(float* p, const float* f) {
        const V4 v = {f[0], f[1], f[2], f[3]};
        __builtin_nontemporal_store(v, (V4*)p);
    }
    static __device__ __forceinline__ float one(const float* p) { return *p; }
    static __device__ __forceinline__ void put(float* p, float f) { *p = f; }
};

// The part of a row that a block takes: vectors k0 .. k1 - 1 and, if it takes
// the last ones, the V % E values past them.
struct Span {
    int k0, k1, i0, i1;
};
template <typename T>
__device__ __forceinline__ Span span_of(int V, int z, int splits) {
    constexpr int E = Row<T>::E;
    const int nv = V / E, per = (nv + splits - 1) / splits;
    const int k0 = min(z * per, nv), k1 = min(k0 + per, nv);
    return {k0, k1, nv * E, z == splits - 1 ? V : nv * E};
}

// statistics of a span over a block of NW waves
template <typename T, int NW, bool ENT, bool NT>
__device__ __forceinline__ SoftRow span_soft_ld(const T* L, const Span& sp, const ExpScale& c2,
                                                float* redm, double (*red)[2]) {
    constexpr int E = Row<T>::E;
    Soft st = {-INFINITY, 0.f, 0.f};
    // (BF16: two vectors in flight a thread, us: 4096 x 151,936 137 -> 134; not for
    // F32 vectors, half as much work each: rows of 50,257 67.4 -> 69.2)
    constexpr int U = E == 8 ? 2 : 1;
#pragma unroll U
    for (int k = sp.k0 + (int)threadIdx.x; k < sp.k1; k += 64 * NW) {
        float f[E];
        Row<T>::unpack(Row<T>::template ld<NT>(L + (int64_t)k * E), f);
        soft_add<E, ENT>(st, f, c2);
    }
    for (int i = sp.i0 + (int)threadIdx.x; i < sp.i1; i += 64 * NW) {
        const float f = Row<T>::one(L + i);
        soft_add<1, ENT>(st, &f, c2);
    }
    return soft_block<NW, ENT>(st, c2.near, redm, red);
}
template <typename T, int NW, bool ENT>
__device__ __forceinline__ SoftRow span_soft(bool nt, const T* L, const Span& sp, const ExpScale& c2,
                                             float* redm, double (*red)[2]) {
    return nt ? span_soft_ld<T, NW, ENT, true>(L, sp, c2, redm, red)
              : span_soft_ld<T, NW, ENT, false>(L, sp, c2, redm, red);
}

// One row per block, each thread's statistics of its vectors joined at the
// end: one read of the rows that have a token, and bound by that (4096 x 151,936
// with 40% of the rows without one: 126 us, 5.8 TB/s).  Holding the row in
// registers gained nothing here: there is no second pass to save.
template <typename T, int NW, bool ENT>
__global__ __launch_bounds__(64 * NW) void k_token_logp(const T* __restrict__ logits, int64_t ld,
                                                        const int32_t* __restrict__ targets,
                                                        float c, ExpScale c2,
                                                        float* __restrict__ logp,
                                                        float* __restrict__ lse,
                                                        float* __restrict__ entropy, int N, int V,
                                                        bool nt) {
    __shared__ float redm[NW];
    __shared__ double red[NW][2];
    const Span sp = span_of<T>(V, 0, 1);
    for (int64_t n = blockIdx.x; n < N; n += gridDim.x) {
        const int t = targets[n];
        RowOut o = {0.0, 0.f, 0.f};
        if (t >= 0) {
            const T* L = logits + n * ld;
            const SoftRow st = span_soft<T, NW, ENT>(nt, L, sp, c2, redm, red);
            if (threadIdx.x == 0) o = row_out(st, t < V ? Row<T>::one(L + t) : 0.f, t < V, c);
        }
        if (threadIdx.x == 0) {
            logp[n] = (float)o.logp;
            lse[n] = o.lse;
            if (ENT) entropy[n] = o.ent;
        }
    }
}

// ── gradient of the logits ──────────────────────────────────────────────
// One logit's gradient without the token's own term c g:
// -c p (g + e (log p + H))
template <bool ENT>
__device__ __forceinline__ float logit_grad(float f, float c, float lse, float H, float g,
                                            float e) {
    const float lp = fmaf(c, f, -lse), p = __builtin_amdgcn_exp2f(lp * kLog2e);
    return -c * (p * (ENT ? fmaf(e, fmaxf(lp, kFar) + H, g) : g));
}
// what a row's gradient takes: the token, lse, entropy, dlogp, dentropy
struct GradRow {
    int t;
    float c, lse, H, g, e;
};
// the same for every lane: taken to scalar registers
__device__ __forceinline__ float uniform_f(float f) {
    return __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(f)));
}
__device__ __forceinline__ GradRow uniform_row(const GradRow& r) {
    return {__builtin_amdgcn_readfirstlane(r.t), uniform_f(r.c), uniform_f(r.lse),
            uniform_f(r.H),                      uniform_f(r.g), uniform_f(r.e)};
}
template <typename T, bool NT>
__device__ __forceinline__ void span_grad_ld(const T* L, T* D, const Span& sp, const GradRow& r,
                                             int tid, int nt) {
    constexpr int E = Row<T>::E;
    for (int k = sp.k0 + tid; k < sp.k1; k += nt) {
        float f[E];
        Row<T>::unpack(Row<T>::template ld<NT>(L + (int64_t)k * E), f);
#pragma unroll
        for (int q = 0; q < E; q++)
            f[q] = logit_grad<true>(f[q], r.c, r.lse, r.H, r.g, r.e) +
                   (k * E + q == r.t ? r.c * r.g : 0.f);
        Row<T>::store(D + (int64_t)k * E, f);
    }
    for (int i = sp.i0 + tid; i < sp.i1; i += nt)
        Row<T>::put(D + i, logit_grad<true>(Row<T>::one(L + i), r.c, r.lse, r.H, r.g, r.e) +
                               (i == r.t ? r.c * r.g : 0.f));
}
template <typename T>
__device__ __forceinline__ void span_grad(bool past, const T* L, T* D, const Span& sp,
                                          const GradRow& r, int tid, int nt) {
    if (past)
        span_grad_ld<T, true>(L, D, sp, r, tid, nt);
    else
        span_grad_ld<T, false>(L, D, sp, r, tid, nt);
}
template <typename T>
__device__ __forceinline__ void span_zero(T* D, const Span& sp, int tid, int nt) {
    constexpr int E = Row<T>::E;
    float z[E];
#pragma unroll
    for (int q = 0; q < E; q++) z[q] = 0.f;
    for (int k = sp.k0 + tid; k < sp.k1; k += nt) Row<T>::store(D + (int64_t)k * E, z);
    for (int i = sp.i0 + tid; i < sp.i1; i += nt) Row<T>::put(D + i, 0.f);
}

// `splits` blocks per row (blockDim.x threads each).  Reads and writes each
// logit once, and bound by that: 2048 x 152,064 of which a quarter have no
// token in 195 us, 5.6 TB/s.
template <typename T>
__global__ __launch_bounds__(512) void k_token_logp_bwd(
    const T* logits, int64_t ld, const int32_t* __restrict__ targets, float c,
    const float* __restrict__ lse, const float* __restrict__ entropy,
    const float* __restrict__ dlogp, const float* __restrict__ dentropy, T* dlogits, int64_t ldd,
    int N, int V, int splits, bool nt) {
    for (int64_t b = blockIdx.x; b < (int64_t)N * splits; b += gridDim.x) {
        const int64_t n = b / splits;
        const Span sp = span_of<T>(V, (int)(b - n * splits), splits);
        GradRow r = {targets[n], c, 0.f, 0.f, 0.f, 0.f};
        if (r.t >= 0) {
            r.g = dlogp[n];
            if (dentropy) r.e = dentropy[n];
        }
        T* D = dlogits + n * ldd;
        if (r.g == 0.f && r.e == 0.f) {
            span_zero(D, sp, threadIdx.x, blockDim.x);
            continue;
        }
        r.lse = lse[n];
        if (r.e != 0.f) r.H = entropy[n];
        span_grad(nt, logits + n * ld, D, sp, r, threadIdx.x, blockDim.x);
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
// exp(d) - d - 1 without its cancellation at the small d of a policy close to
// its reference
__device__ __forceinline__ double kl_d(double d) {
    if (fabs(d) > 0.5) return exp_d(d) - 1.0 - d;
    double p = 1.0 / 479001600.0;
    p = fma(p, d, 1.0 / 39916800.0);
    p = fma(p, d, 1.0 / 3628800.0);
    p = fma(p, d, 1.0 / 362880.0);
    p = fma(p, d, 1.0 / 40320.0);
    p = fma(p, d, 1.0 / 5040.0);
    p = fma(p, d, 1.0 / 720.0);
    p = fma(p, d, 1.0 / 120.0);
    p = fma(p, d, 1.0 / 24.0);
    p = fma(p, d, 1.0 / 6.0);
    return d * d * fma(p, d, 0.5);
}
// In 64 bits, from the logp before its rounding to F32.
__device__ __forceinline__ PolicyTok policy_token(const PolicyArgs& a, int64_t n, double logp,
                                                  float ent, float w) {
    const double A = a.adv[n];
    double lr = a.old_logp ? logp - (double)a.old_logp[n] : 0.0;
    const bool far = !(fabs(lr) <= 60.0);
    if (far) lr = lr > 0 ? 60.0 : lr < 0 ? -60.0 : lr;
    const double r = exp_d(lr), hi = 1.0 + (double)a.hi, lo = 1.0 - (double)a.lo;
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
        double d = (double)a.ref_logp[n] - logp;
        const bool farr = !(fabs(d) <= 60.0);
        if (farr) d = d > 0 ? 60.0 : d < 0 ? -60.0 : d;
        kl = kl_d(d);
        nan += d - d;
        if (!farr) g -= (double)a.kl_beta * (kl + d);
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

// ── policy step over rows of logits ─────────────────────────────────────
struct PolicyRows {
    const bf16* logits;
    int64_t ld;
    const int32_t* targets;
    float c;
    ExpScale c2;
    float *logp, *entropy, *loss, *kl;
    bf16* dlogits;
    int64_t ldd;
    int N, V;
    bool nt;
};
// a row's weight: 0 where it has no token
__device__ __forceinline__ float row_weight(const PolicyRows& r, const PolicyArgs& a, int64_t n) {
    return r.targets[n] >= 0 ? a.weight[n] : 0.f;
}
// the row's results, and what its gradient takes
__device__ __forceinline__ GradRow policy_row(const PolicyRows& r, const PolicyArgs& a, int64_t n,
                                              const SoftRow& st, float ft, float w) {
    const int t = r.targets[n];
    const RowOut o = row_out(st, ft, t < r.V, r.c);
    const float H = r.entropy ? o.ent : 0.f;
    const PolicyTok pt = policy_token(a, n, o.logp, H, w);
    r.logp[n] = (float)o.logp;
    if (r.entropy) r.entropy[n] = H;
    r.loss[n] = pt.loss;
    if (r.kl) r.kl[n] = pt.kl;
    return {t, r.c, o.lse, H, pt.dlogp, -a.ent_coef * w};
}
__device__ __forceinline__ void policy_no_row(const PolicyRows& r, int64_t n) {
    r.logp[n] = 0.f;
    if (r.entropy) r.entropy[n] = 0.f;
    r.loss[n] = 0.f;
    if (r.kl) r.kl[n] = 0.f;
}

// Two passes over the row, the second out of the caches: for rows too long for
// a block's registers (2048 x 151,936, a quarter without a token: 280 us, 233
// in registers).
template <bool ENT>
__global__ __launch_bounds__(512) void k_policy_logits(PolicyRows r, PolicyArgs a) {
    __shared__ float redm[8];
    __shared__ double red[8][2];
    __shared__ GradRow sg;
    const Span sp = span_of<bf16>(r.V, 0, 1);
    for (int64_t n = blockIdx.x; n < r.N; n += gridDim.x) {
        const float w = row_weight(r, a, n);
        const bf16* L = r.logits + n * r.ld;
        bf16* D = r.dlogits + n * r.ldd;
        if (w != 0.f) {
            const int t = r.targets[n];
            const float ft = t < r.V ? bf2f(L[t]) : 0.f;
            const SoftRow st = span_soft<bf16, 8, ENT>(r.nt, L, sp, r.c2, redm, red);
            if (threadIdx.x == 0) sg = policy_row(r, a, n, st, ft, w);
            __syncthreads();
            span_grad(r.nt, L, D, sp, sg, threadIdx.x, 512);
        } else {
            span_zero(D, sp, threadIdx.x, 512);
            if (threadIdx.x == 0) policy_no_row(r, n);
        }
        __syncthreads();  // sg is read before the next row writes it
    }
}

// A row held in the registers of its block of NT threads, so that it is read
// once: up to CPT whole sweeps of NT vectors, the part sweep after them and the
// V % E values past the vectors (CPT <= 19 of BF16: 80 registers of a lane,
// where a 1024-thread block has 128).  Whether a sweep is whole is the same for
// every lane, so it costs no lane mask and one address register for all.
template <typename T, int CPT, int NT>
struct RegRow {
    typedef typename Row<T>::V4 V4;
    static constexpr int E = Row<T>::E;
    V4 v[CPT], vp;
    float ft;
    int whole, part;  // whole sweeps, vectors of the part sweep
    int tail;         // index of this lane's value past the vectors, or -1
    __device__ __forceinline__ void load(const T* L, int V, bool nt) {
        const int nv = V / E, it = nv * E + (int)threadIdx.x;
        whole = nv / NT;
        part = nv % NT;
        tail = it < V ? it : -1;
        if (nt) {
#pragma unroll
            for (int k = 0; k < CPT; k++)
                if (k < whole)
                    v[k] = Row<T>::template ld<true>(L + (int64_t)k * NT * E + threadIdx.x * E);
        } else {
#pragma unroll
            for (int k = 0; k < CPT; k++)
                if (k < whole)
                    v[k] = Row<T>::template ld<false>(L + (int64_t)k * NT * E + threadIdx.x * E);
        }
        if ((int)threadIdx.x < part)
            vp = Row<T>::template ld<false>(L + (int64_t)whole * NT * E + threadIdx.x * E);
        ft = tail >= 0 ? Row<T>::one(L + tail) : 0.f;
    }
    // f(values, first index) for every vector of the lane.  The empty asm
    // statement makes each pass unpack anew: kept unpacked from one pass to
    // the next, a row takes 160 registers and spills.
    template <typename F>
    __device__ __forceinline__ void each(F&& f) {
#pragma unroll
        for (int k = 0; k < CPT; k++)
            if (k < whole) {
                asm volatile("" : "+v"(v[k]));
                float x[E];
                Row<T>::unpack(v[k], x);
                f(x, k * NT + (int)threadIdx.x, k);
                __builtin_amdgcn_sched_barrier(0);  // one vector's temporaries at a time
            }
        if ((int)threadIdx.x < part) {
            asm volatile("" : "+v"(vp));
            float x[E];
            Row<T>::unpack(vp, x);
            f(x, whole * NT + (int)threadIdx.x, whole);
        }
    }
    template <bool ENT>
    __device__ __forceinline__ SoftRow soft(const ExpScale& c2, float* redm, double (*red)[2]) {
        float m = tail >= 0 ? ft : -INFINITY;
        each([&](const float* x, int, int) {
#pragma unroll
            for (int e = 0; e < E; e++) m = fmaxf(m, x[e]);
        });
        m = block_maxf<NT / 64>(m, redm);
        const float R = soft_ref(m);
        float s = 0.f, u = 0.f;
        auto add = [&](float x, float& s, float c2) {
            const float d = x - R, p = __builtin_amdgcn_exp2f(d * c2);
            s += p;
            if (ENT) u = fmaf(p, fmaxf(d, kFar), u);
        };
        if (tail >= 0) add(ft, s, c2.near);
        each([&](const float* x, int, int) {
            float sv = 0.f;
#pragma unroll
            for (int e = 0; e < E; e++) add(x[e], sv, c2.c[e]);
            s += sv;
        });
        return block_sums<NT / 64, ENT>(m, s, u, red);
    }
};

// The policy step of one row, read once and written once: statistics, loss and
// dlogp of the token by one thread, gradient.  Bound by the two streams (2048 x
// 151,936, a quarter of the rows without a token, KL term and entropy: 234 us,
// 4.4 TB/s, 0.95 of a large copy's rate).
template <int CPT, int NT, bool ENT>
__global__ __launch_bounds__(NT) void k_policy_reg(PolicyRows r, PolicyArgs a) {
    __shared__ float redm[NT / 64];
    __shared__ double red[NT / 64][2];
    __shared__ GradRow sg;
    const int64_t n = blockIdx.x;
    const float w = row_weight(r, a, n);
    const bf16* L = r.logits + n * r.ld;
    bf16* D = r.dlogits + n * r.ldd;
    if (w == 0.f) {
        span_zero(D, span_of<bf16>(r.V, 0, 1), threadIdx.x, NT);
        if (threadIdx.x == 0) policy_no_row(r, n);
        return;
    }
    // (every load of the row is before the block's barriers, which the stores
    // to dlogits, maybe the same row, are behind)
    RegRow<bf16, CPT, NT> row;
    row.load(L, r.V, r.nt);
    const int t = r.targets[n];
    const float ft = t < r.V ? bf2f(L[t]) : 0.f;
    const SoftRow st = row.template soft<ENT>(r.c2, redm, red);
    if (threadIdx.x == 0) sg = policy_row(r, a, n, st, ft, w);
    __syncthreads();
    const GradRow g = uniform_row(sg);
    const int tc = g.t >> 3;
    row.each([&](const float* x, int q, int k) {
        float f[8];
#pragma unroll
        for (int i = 0; i < 8; i++) f[i] = logit_grad<ENT>(x[i], g.c, g.lse, g.H, g.g, g.e);
        if (q == tc) {
#pragma unroll
            for (int i = 0; i < 8; i++) f[i] += i == (g.t & 7) ? g.c * g.g : 0.f;
        }
        Row<bf16>::store(D + (int64_t)k * NT * 8 + 8 * threadIdx.x, f);
    });
    if (row.tail >= 0)
        D[row.tail] = f2bf(logit_grad<ENT>(row.ft, g.c, g.lse, g.H, g.g, g.e) +
                           (row.tail == g.t ? g.c * g.g : 0.f));
}

// ── few rows: each over several blocks ──────────────────────────────────
// See row_splits; part [N][splits] statistics.  One row of 151,936: 3.6 us for
// the parts and 2.2 to join them, where one block draws the row in 11.
template <typename T, bool ENT>
__global__ __launch_bounds__(512) void k_soft_part(const T* __restrict__ logits, int64_t ld,
                                                   const int32_t* __restrict__ targets,
                                                   const float* __restrict__ weight, ExpScale c2,
                                                   SoftRow* __restrict__ part, int V, int splits) {
    __shared__ float redm[8];
    __shared__ double red[8][2];
    const int64_t n = blockIdx.x / splits;
    const int z = (int)(blockIdx.x - n * splits);
    if (targets[n] < 0 || (weight && weight[n] == 0.f)) return;
    const SoftRow st =
        span_soft<T, 8, ENT>(false, logits + n * ld, span_of<T>(V, z, splits), c2, redm, red);
    if (threadIdx.x == 0) part[blockIdx.x] = st;
}
// a row's statistics from its parts (splits <= 64), by one wave
template <bool ENT>
__device__ __forceinline__ SoftRow parts_merge(const SoftRow* part, int64_t n, int splits,
                                               float c2) {
    const int lane = threadIdx.x & 63;
    SoftRow p = {-INFINITY, 0.0, 0.0};
    if (lane < splits) p = part[n * splits + lane];
    const float m = wave_max(p.m), d = p.m - soft_ref(m);
    const double f = (double)__builtin_amdgcn_exp2f(d * c2);
    return {m, wave_sum_d(f * p.s),
            ENT ? wave_sum_d(f * (p.u + p.s * (double)fmaxf(d, kFar))) : 0.0};
}
template <typename T, bool ENT>
__global__ __launch_bounds__(64) void k_token_logp_join(const T* __restrict__ logits, int64_t ld,
                                                        const int32_t* __restrict__ targets,
                                                        float c, const SoftRow* __restrict__ part,
                                                        int splits, float* __restrict__ logp,
                                                        float* __restrict__ lse,
                                                        float* __restrict__ entropy, int V) {
    const int64_t n = blockIdx.x;
    const int t = targets[n];
    RowOut o = {0.0, 0.f, 0.f};
    if (t >= 0)
        o = row_out(parts_merge<ENT>(part, n, splits, c * kLog2e),
                    t < V ? Row<T>::one(logits + n * ld + t) : 0.f, t < V, c);
    if (threadIdx.x != 0) return;
    logp[n] = (float)o.logp;
    lse[n] = o.lse;
    if (ENT) entropy[n] = o.ent;
}
template <bool ENT>
__global__ __launch_bounds__(64) void k_policy_join(PolicyRows r, PolicyArgs a,
                                                    const SoftRow* __restrict__ part, int splits,
                                                    GradRow* __restrict__ grads) {
    const int64_t n = blockIdx.x;
    const float w = row_weight(r, a, n);
    GradRow g = {-1, r.c, 0.f, 0.f, 0.f, 0.f};
    if (w != 0.f) {
        const SoftRow st = parts_merge<ENT>(part, n, splits, r.c * kLog2e);
        const int t = r.targets[n];
        const float ft = t < r.V ? bf2f(r.logits[n * r.ld + t]) : 0.f;
        if (threadIdx.x == 0) g = policy_row(r, a, n, st, ft, w);
    } else if (threadIdx.x == 0) {
        policy_no_row(r, n);
    }
    if (threadIdx.x == 0) grads[n] = g;
}
__global__ __launch_bounds__(512) void k_policy_grad(PolicyRows r,
                                                     const GradRow* __restrict__ grads,
                                                     int splits) {
    const int64_t n = blockIdx.x / splits;
    const Span sp = span_of<bf16>(r.V, (int)(blockIdx.x - n * splits), splits);
    const GradRow g = grads[n];
    bf16* D = r.dlogits + n * r.ldd;
    if (g.t >= 0)
        span_grad(false, r.logits + n * r.ld, D, sp, g, threadIdx.x, 512);
    else
        span_zero(D, sp, threadIdx.x, 512);
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
// log(1 + e) for 0 <= e <= 1
__device__ __forceinline__ double log1p_d(double e) {
    if (e > 1.0 / 128) return log_d(1.0 + e);
    return e * fma(e, fma(e, fma(e, fma(e, 0.2, -0.25), 1.0 / 3), -0.5), 1.0);
}
// (-|z| past 700: exp is 0 beside the first term in any precision here)
__device__ __forceinline__ double exp_neg(double z) { return exp_d(fmax(-fabs(z), -700.0)); }
__device__ __forceinline__ double softplus(double z) { return fmax(z, 0.0) + log1p_d(exp_neg(z)); }
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
    if (u != u) {  // (the maxima and tests below drop a NaN)
        *loss = u;
        return u;
    }
    if (a.kind == TA_PREF_SIGMOID) {
        *loss = (1.0 - sm) * softplus(-z) + sm * softplus(z);
        // sigma(z) - (1 - smoothing), without cancelling at large z
        const double e = exp_neg(z), tail = e / (1.0 + e);
        du = beta * (z >= 0 ? sm - tail : tail - (1.0 - sm));
    } else if (a.kind == TA_PREF_IPO) {
        const double v = u - (double)a.margin - 1.0 / (2.0 * beta);
        *loss = v * v;
        du = 2.0 * v;
    } else {
        *loss = fmax(1.0 - z, 0.0);
        du = z < 1.0 ? -beta : 0.0;
    }
    return du * (double)a.scale;
}
__device__ __forceinline__ int64_t wave_sum_l(int64_t v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
    return v;
}

// four tokens' values, at any address of their type
template <typename T>
struct Tok4 {
    typedef T V __attribute__((ext_vector_type(4), aligned(4)));
};
// One block of NW waves per pair: half of them sum the chosen answer, half
// the rejected one, then the loss, then the gradient.  Bound by latency: a
// launch, one or a few loads in a row, the loss of one thread (4 pairs of 300
// tokens 3.7 us, where an empty launch takes 2.9).
template <int NW>
__global__ __launch_bounds__(64 * NW) void k_preference(PrefArgs a) {
    constexpr int NH = NW / 2, NT = 64 * NH;
    __shared__ double sp[NW], sr[NW], sg[2];
    __shared__ int64_t sc[NW];
    const int64_t p = blockIdx.x;
    const int w = threadIdx.x >> 6, side = w >= NH, tid = threadIdx.x - side * NT;
    const int64_t b = min(max(a.offsets[2 * p + side], (int64_t)0), a.N);
    const int64_t e = min(max(a.offsets[2 * p + side + 1], b), a.N);
    double pi = 0.0, rf = 0.0;
    int64_t cnt = 0;
    // (values of tokens that do not count are loaded and left out, so the
    // loads do not wait for the targets)
    auto add = [&](int t, float l, float r) {
        const bool on = t >= 0;
        pi += on ? (double)l : 0.0;
        rf += on ? (double)r : 0.0;
        cnt += on;
    };
    const int64_t e4 = b + (e - b) / 4 * 4;  // four tokens a thread, then the rest
#pragma unroll 2
    for (int64_t j = b + 4 * tid; j < e4; j += 4 * NT) {
        const Tok4<int32_t>::V t = *(const Tok4<int32_t>::V*)(a.targets + j);
        const Tok4<float>::V l = *(const Tok4<float>::V*)(a.logp + j);
        Tok4<float>::V r = {0.f, 0.f, 0.f, 0.f};
        if (a.ref) r = *(const Tok4<float>::V*)(a.ref + j);
#pragma unroll
        for (int i = 0; i < 4; i++) add(t[i], l[i], r[i]);
    }
    if (e4 + tid < e) add(a.targets[e4 + tid], a.logp[e4 + tid], a.ref ? a.ref[e4 + tid] : 0.f);
    pi = wave_sum_d(pi);
    rf = wave_sum_d(rf);
    cnt = wave_sum_l(cnt);
    if ((threadIdx.x & 63) == 0) sp[w] = pi, sr[w] = rf, sc[w] = cnt;
    __syncthreads();
    if (threadIdx.x == 0) {
        PrefSums q;
        for (int i = 0; i < 2; i++) {
            q.pi[i] = sp[i * NH], q.rf[i] = sr[i * NH], q.cnt[i] = sc[i * NH];
            for (int k = 1; k < NH; k++)
                q.pi[i] += sp[i * NH + k], q.rf[i] += sr[i * NH + k], q.cnt[i] += sc[i * NH + k];
        }
        double loss, rew[2];
        const double du = pref_pair(a, q, &loss, rew);
        for (int i = 0; i < 2; i++)
            sg[i] = (i ? -du : du) * (a.average && q.cnt[i] > 0 ? 1.0 / (double)q.cnt[i] : 1.0);
        a.pair_loss[p] = (float)loss;
        if (a.rewards) {
            a.rewards[2 * p] = (float)rew[0];
            a.rewards[2 * p + 1] = (float)rew[1];
        }
    }
    __syncthreads();
    if (!a.dlogp) return;
    const float g = (float)sg[side];
#pragma unroll 2
    for (int64_t j = b + 4 * tid; j < e4; j += 4 * NT) {
        const Tok4<int32_t>::V t = *(const Tok4<int32_t>::V*)(a.targets + j);
        const Tok4<float>::V d = {t[0] >= 0 ? g : 0.f, t[1] >= 0 ? g : 0.f, t[2] >= 0 ? g : 0.f,
                                  t[3] >= 0 ? g : 0.f};
        *(Tok4<float>::V*)(a.dlogp + j) = d;
    }
    if (e4 + tid < e) a.dlogp[e4 + tid] = a.targets[e4 + tid] >= 0 ? g : 0.f;
}

// at most this many blocks of a launch over rows (its threads stay below 2^32)
static inline dim3 row_grid(int64_t rows) {
    return dim3((unsigned)std::min<int64_t>(rows, 1 << 20));
}
constexpr int kMaxV = 1 << 30;  // indices into a row stay below 2^31
static bool temp_ok(float c) { return c > 0.f && c < INFINITY; }

// Waves of a row's block in the forward: narrow ones where the row has hardly a
// vector per lane of eight waves, and where there are many rows to share a CU
// (us, 2 / 4 / 8 waves: 2000 rows of 1000 4.2 / 5.2 / 7.9, of 8000 11.0 / 9.8 /
// 11.7; 100 rows of 8000 5.6 / 4.4 / 3.9).
static int fwd_waves(int N, int V) {
    return V <= 2048 ? 2 : V <= 4096 || (V <= 12288 && N >= 512) ? 4 : 8;
}
// Threads of a gradient's block (128 / 256 / 512, us: 2000 rows of 1000 4.2 /
// 4.9 / 6.4, of 4000 9.0 / 8.4 / 8.8, of 8000 15.3 / 14.6 / 13.7).
static int bwd_threads(int V) { return V <= 1024 ? 128 : V <= 4096 ? 256 : 512; }

// Blocks that each row's statistics are split over (1: one block per row,
// also in a capture, where graphs of one stream would share the parts).  One
// CU draws about 25 KB a microsecond of rows that are not in its L2, so up to
// max_rows rows of 192 KB or more are faster in parts that are joined by a
// second launch (151,936 BF16, cold, us with the host's launches: 1 row 17 ->
// 11, 64 rows 26 -> 11, 384 rows 33 -> 26; 65,536 8 -> 11).
static int row_splits(int N, int V, int es, int max_rows, hipStream_t s) {
    if (N > max_rows || (int64_t)V * es < (192 << 10) || is_capturing(s)) return 1;
    const int64_t sweeps = (int64_t)V * es / (512 * 16);
    return (int)std::min<int64_t>({sweeps, 64, std::max(1024 / N, 2)});
}
// Blocks per row of the gradient: a thousand in all, a sweep of vectors each
// at least.
static int grad_splits(int N, int V, int es) {
    const int64_t sweeps = (int64_t)V * es / (512 * 16);
    return (int)std::max<int64_t>(1, std::min<int64_t>(sweeps, 1024 / N));
}

template <typename T>
static int token_logp_fwd(const T* logits, int64_t ld, const int32_t* targets, float c, float* logp,
                          float* lse, float* entropy, int N, int V, hipStream_t s) {
    TA_REQUIRE(N >= 0 && V > 0 && V <= kMaxV && ld >= V,
               "token_logp_fwd: bad shape N=%d V=%d ld=%lld", N, V, (long long)ld);
    TA_REQUIRE(temp_ok(c), "token_logp_fwd: inv_temp must be positive and finite");
    if (N == 0) return 0;
    TA_REQUIRE(logits && targets && logp && lse, "token_logp_fwd: null argument");
    TA_REQUIRE(((uintptr_t)logits % sizeof(T)) == 0, "token_logp_fwd: misaligned logits");
    const int splits = row_splits(N, V, sizeof(T), 512, s);
    if (splits > 1) {
        SoftRow* part = nullptr;
        if (int rc = scratch_here("token_logp_fwd", sizeof(SoftRow) * N * splits, s, (void**)&part))
            return rc;
        const dim3 grid(N * splits);
        const float* no_weight = nullptr;
        if (entropy) {
            tlaunch(k_soft_part<T, true>, grid, dim3(512), s, logits, ld, targets, no_weight,
                    exp_scale(c), part, V, splits);
            tlaunch(k_token_logp_join<T, true>, dim3(N), dim3(64), s, logits, ld, targets, c, part,
                    splits, logp, lse, entropy, V);
        } else {
            tlaunch(k_soft_part<T, false>, grid, dim3(512), s, logits, ld, targets, no_weight,
                    exp_scale(c), part, V, splits);
            tlaunch(k_token_logp_join<T, false>, dim3(N), dim3(64), s, logits, ld, targets, c,
                    part, splits, logp, lse, entropy, V);
        }
        return check_launch("token_logp_fwd");
    }
    const bool nt = (int64_t)N * V * (int64_t)sizeof(T) > kCacheBytes;
    const ExpScale c2 = exp_scale(c);
#define TL(NW, ENT)                                                                             \
    tlaunch(k_token_logp<T, NW, ENT>, row_grid(N), dim3(64 * NW), s, logits, ld, targets, c, c2, \
            logp, lse, entropy, N, V, nt)
    const int nw = fwd_waves(N, V);
    if (nw == 2) {
        if (entropy) TL(2, true);
        else TL(2, false);
    } else if (nw == 4) {
        if (entropy) TL(4, true);
        else TL(4, false);
    } else {
        if (entropy) TL(8, true);
        else TL(8, false);
    }
#undef TL
    return check_launch("token_logp_fwd");
}

template <typename T>
static int token_logp_bwd(const T* logits, int64_t ld, const int32_t* targets, float c,
                          const float* lse, const float* entropy, const float* dlogp,
                          const float* dentropy, T* dlogits, int64_t ldd, int N, int V,
                          hipStream_t s) {
    TA_REQUIRE(N >= 0 && V > 0 && V <= kMaxV && ld >= V && ldd >= V,
               "token_logp_bwd: bad shape N=%d V=%d ld=%lld ldd=%lld", N, V, (long long)ld,
               (long long)ldd);
    TA_REQUIRE(temp_ok(c), "token_logp_bwd: inv_temp must be positive and finite");
    if (N == 0) return 0;
    TA_REQUIRE(logits && targets && lse && dlogp && dlogits, "token_logp_bwd: null argument");
    TA_REQUIRE(!dentropy || entropy, "token_logp_bwd: dentropy needs the entropy");
    TA_REQUIRE((((uintptr_t)logits | (uintptr_t)dlogits) % sizeof(T)) == 0,
               "token_logp_bwd: misaligned rows");
    TA_REQUIRE(dlogits != logits || ldd == ld, "token_logp_bwd: in place needs ldd = ld");
    const int splits = grad_splits(N, V, sizeof(T));
    tlaunch(k_token_logp_bwd<T>, row_grid((int64_t)N * splits), dim3(bwd_threads(V)), s,
            logits, ld, targets, c, lse, entropy, dlogp, dentropy, dlogits, ldd, N, V, splits,
            (int64_t)N * V * (int64_t)sizeof(T) > kCacheBytes);
    return check_launch("token_logp_bwd");
}

int policy_config_check(const char* what, float lo, float hi, float dual, float kl_beta,
                        float ent_coef, float inv_temp) {
    TA_REQUIRE(temp_ok(inv_temp), "%s: inv_temp must be positive and finite", what);
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
    TA_REQUIRE(fabsf(margin) < INFINITY && fabsf(scale) < INFINITY,
               "preference_loss: margin and scale must be finite");
    if (P == 0) return 0;
    TA_REQUIRE(offsets && pair_loss && (N == 0 || (logp && targets)),
               "preference_loss: null argument");
    const PrefArgs a{logp,      ref_logp, targets, offsets, N,         kind,    average, beta,
                     smoothing, margin,   scale,   pair_loss, rewards, dlogp};
    // (4 / 16 waves, us: answers of 1000 tokens 4.1 / 4.3, of 2000 4.9 / 4.7, of
    // 16,000 13.8 / 9.2)
    if (N / P > 2048)
        tlaunch(k_preference<16>, dim3(P), dim3(1024), (hipStream_t)stream, a);
    else
        tlaunch(k_preference<4>, dim3(P), dim3(256), (hipStream_t)stream, a);
    return check_launch("preference_loss");
}

int ta_policy_loss(const float* logp, const float* old_logp, const float* ref_logp,
                   const float* adv, const float* weight, float clip_lo, float clip_hi,
                   float dual_clip, float kl_beta, float* loss, float* kl, float* dlogp,
                   int64_t N, void* stream) {
    TA_REQUIRE(N >= 0, "policy_loss: bad shape N=%lld", (long long)N);
    if (N == 0) return 0;
    TA_REQUIRE(logp && adv && weight && dlogp, "policy_loss: null argument");
    if (int rc = policy_config_check("policy_loss", clip_lo, clip_hi, dual_clip, kl_beta, 0.f, 1.f))
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
    TA_REQUIRE(N >= 0 && V > 0 && V <= kMaxV && ld >= V && ldd >= V,
               "policy_loss_logits: bad shape N=%d V=%d ld=%lld ldd=%lld", N, V, (long long)ld,
               (long long)ldd);
    if (int rc = policy_config_check("policy_loss_logits", clip_lo, clip_hi, dual_clip, kl_beta,
                                     ent_coef, inv_temp))
        return rc;
    if (N == 0) return 0;
    TA_REQUIRE(logits && targets && adv && weight && logp && loss && dlogits,
               "policy_loss_logits: null argument");
    TA_REQUIRE(ent_coef == 0.f || entropy, "policy_loss_logits: ent_coef needs the entropy");
    TA_REQUIRE((((uintptr_t)logits | (uintptr_t)dlogits) & 1) == 0,
               "policy_loss_logits: misaligned rows");
    TA_REQUIRE(dlogits != logits || ldd == ld, "policy_loss_logits: in place needs ldd = ld");
    const PolicyArgs a{old_logp, ref_logp, adv,       weight,  clip_lo,
                       clip_hi,  dual_clip, kl_beta, ent_coef};
    hipStream_t s = (hipStream_t)stream;
    const PolicyRows r{logits, ld,   targets, inv_temp, exp_scale(inv_temp), logp, entropy,
                       loss,   kl,   dlogits, ldd,      N,    V,
                       (int64_t)N * V * 2 > kCacheBytes};
    // (three launches instead of one: 1 row of 151,936 26 -> 15 us, 64 rows 30
    // -> 20, 128 rows 31 -> 30)
    const int splits = row_splits(N, V, 2, 96, s);
    if (splits > 1) {
        const size_t gb = ((size_t)N * sizeof(GradRow) + 255) & ~(size_t)255;
        char* ws = nullptr;
        if (int rc = scratch_here("policy_loss_logits", gb + sizeof(SoftRow) * N * splits, s,
                                  (void**)&ws))
            return rc;
        GradRow* grads = (GradRow*)ws;
        SoftRow* part = (SoftRow*)(ws + gb);
        const dim3 grid(N * splits);
        if (entropy) {
            tlaunch(k_soft_part<bf16, true>, grid, dim3(512), s, logits, ld, targets, weight,
                    exp_scale(inv_temp), part, V, splits);
            tlaunch(k_policy_join<true>, dim3(N), dim3(64), s, r, a, part, splits, grads);
        } else {
            tlaunch(k_soft_part<bf16, false>, grid, dim3(512), s, logits, ld, targets, weight,
                    exp_scale(inv_temp), part, V, splits);
            tlaunch(k_policy_join<false>, dim3(N), dim3(64), s, r, a, part, splits, grads);
        }
        tlaunch(k_policy_grad, grid, dim3(512), s, r, grads, splits);
        return check_launch("policy_loss_logits");
    }
    // Rows in registers: the narrowest block that holds the row lets the most
    // rows share a CU, whose loads, sums and stores then overlap (2000 rows, us,
    // blocks of 128 / 256 / 512 / 1024 threads: of 1000 logits 6.6 / 8.3 / 12.6 /
    // 22.7, of 16,000 30 / 30 / 30 / 38, of 40,000 - / 66 / 71 / 90, of 80,000 - /
    // - / 127 / 157); few rows are faster in wider ones (100 of 16,000 10.3 / 7.7
    // / 7.4 / 7.6).
    const int nt = V <= 2048                                ? 128
                   : V <= 8192 || (V < 40960 && N >= 1000) ? 256
                   : V < 81920                              ? 512
                                                            : 1024;
    const int sweeps = V / 8 / nt;
    if (sweeps <= 19 && N <= (1 << 20)) {
#define PL(C, NT)                                                           \
    do {                                                                    \
        if (entropy)                                                        \
            tlaunch(k_policy_reg<C, NT, true>, dim3(N), dim3(NT), s, r, a); \
        else                                                                \
            tlaunch(k_policy_reg<C, NT, false>, dim3(N), dim3(NT), s, r, a); \
    } while (0)
#define PL4(NT)                    \
    if (sweeps <= 3) PL(3, NT);    \
    else if (sweeps <= 7) PL(7, NT); \
    else if (sweeps <= 15) PL(15, NT); \
    else PL(19, NT)
        if (nt == 128) {
            PL(3, 128);
        } else if (nt == 256) {
            PL4(256);
        } else if (nt == 512) {
            PL4(512);
        } else if (sweeps <= 15) {
            PL(15, 1024);
        } else {
            PL(19, 1024);
        }
#undef PL4
#undef PL
    } else if (entropy) {
        tlaunch(k_policy_logits<true>, row_grid(N), dim3(512), s, r, a);
    } else {
        tlaunch(k_policy_logits<false>, row_grid(N), dim3(512), s, r, a);
    }
    return check_launch("policy_loss_logits");
}

}  // extern "C"
