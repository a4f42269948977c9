"""Token log-probabilities, LM head scoring, preference loss and policy loss
through the C-ABI against plain implementations in 64 bits.

Tolerances, from the roundings of the kernels (EPS = 2^-24, half a step of
F32): a softmax sum S adds at most V/256 terms one after the other in a lane
and merges a few tens of partial sums; each term exp(c (f - M)) carries the
rounding of its argument, at most |arg| <= 40 for terms that matter, 3
roundings, and the exponential's own step.  So S is within
(V/256 + 64 + 120) EPS; log S and c (f_t - M) add their own roundings.
BF16 results are within half a step, 2^-8 relative, of the F32 value."""
import ctypes
import math

import numpy as np
import pytest
import torch

import tadapt

pytestmark = pytest.mark.gpu

DEV = "cuda"
EPS = 2.0 ** -24
F = ctypes.c_float
P = tadapt.ptr
BF16 = torch.bfloat16
INF, NAN = float("inf"), float("nan")


def S():
    return tadapt.stream()


def call(name, *a):
    tadapt.call(name, *a)


def gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def randn(g, *shape, std=1.0, dtype=torch.float32):
    return (torch.randn(*shape, generator=g, device=DEV) * std).to(dtype)


def rows(g, N, V, dtype, pad=0, std=2.0):
    return randn(g, N, V + pad, std=std, dtype=dtype)[:, :V]


def tokens(g, N, V, masked=0.25):
    t = torch.randint(0, V, (N,), generator=g, device=DEV, dtype=torch.int32)
    off = torch.rand(N, generator=g, device=DEV) < masked
    return torch.where(off, torch.full_like(t, -1), t)


def full(n, v=7.0):
    return torch.full((n,), v, device=DEV)


def ref_logp(x, t, c):
    """(logp, lse, entropy, log p) in float64; masked rows 0."""
    lp = torch.log_softmax(x.double() * c, 1)
    live = (t >= 0).double()
    tl = t.clamp(min=0).long()[:, None]
    lse = (x.double() * c - lp).amax(1) * live
    p = lp.exp()
    ent = -torch.where(p > 0, p * lp, torch.zeros_like(lp)).sum(1) * live
    return lp.gather(1, tl)[:, 0] * live, lse, ent, lp


def sum_tol(V):
    return (V / 256 + 64 + 120) * EPS


def close(got, want, tol, what=""):
    got, want = got.double(), want.double()
    bad = (got - want).abs() > tol
    bad |= torch.isnan(got) != torch.isnan(want)
    assert not bad.any(), (what, int(bad.sum()), float((got - want).abs().max()),
                           float(torch.as_tensor(tol).max()))


def check_fwd(x, t, c, logp, lse, ent):
    V = x.shape[1]
    wl, ws, we, _ = ref_logp(x, t, c)
    span = x.double().abs().amax(1) * c * 2 + math.log(V) + 1
    close(logp, wl, sum_tol(V) + 4 * EPS * span, "logp")
    close(lse, ws, sum_tol(V) + 4 * EPS * span, "lse")
    if ent is not None:
        # log S - c U / S, both at most log V + 1 apart
        close(ent, we, 4 * (math.log(V) + 2) * sum_tol(V), "entropy")


def check_bwd(x, t, c, d, g, e, V):
    wl, ws, we, lp = ref_logp(x, t, c)
    live = (t >= 0).double()[:, None]
    p = lp.exp()
    one = torch.zeros_like(p).scatter_(1, t.clamp(min=0).long()[:, None], 1.0)
    G = g.double()[:, None]
    E = e.double()[:, None] if e is not None else torch.zeros_like(G)
    want = c * (G * (one - p) - E * p * (lp + we[:, None])) * live
    size = c * p * (G.abs() + E.abs() * (lp.abs() + we[:, None] + 1)) * live
    # p from the F32 lse: its argument carries 2 roundings of x, lse and their
    # difference; with the entropy's own error in the second term
    rel = sum_tol(V) + 8 * EPS * (x.double().abs() * c + ws.abs()[:, None] + 4)
    rel = rel + E.abs() / (G.abs() + E.abs() + 1e-30) * 4 * (math.log(V) + 2) * sum_tol(V)
    step = 2.0 ** -8 if d.dtype == BF16 else EPS
    # (results below the normal range flush to zero)
    close(d, want, want.abs() * step * 1.01 + size * rel * 1.01 + c * G.abs() * one * EPS * 2
          + 2.0 ** -125 * (1 + G.abs() + E.abs()) * c, "dlogits")


SHAPES = [(1, 1), (1, 2), (3, 7), (2, 8), (5, 63), (4, 513), (66, 1000), (3, 4104), (2, 20481),
          (5, 50257), (3, 151936), (2, 152064), (2, 163848), (2, 170000), (1, 200003)]


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("N,V", SHAPES)
def test_token_logp(N, V, dtype):
    for k, (pad, c, with_ent, inplace) in enumerate([(0, 1.0, False, False), (13, 0.7, True, False),
                                                     (8, 1.3, True, True), (3, 1.0, False, True)]):
        print(N, V, dtype, pad, c, with_ent, inplace, flush=True)
        g = gen(N * 1000003 + V + k)
        dt, sfx = (BF16, "") if dtype == "bf16" else (torch.float32, "_f32")
        x = rows(g, N, V, dt, pad)
        t = tokens(g, N, V, 0.3 if N > 2 else 0.0)
        logp, lse, ent = full(N), full(N), full(N)
        call("ta_token_logp_fwd" + sfx, P(x), x.stride(0), P(t), F(c), P(logp), P(lse),
             P(ent) if with_ent else None, N, V, S())
        c32 = float(np.float32(c))
        check_fwd(x, t, c32, logp, lse, ent if with_ent else None)
        if not with_ent:
            assert (ent == 7.0).all()
        dl = randn(g, N)
        if N > 3:
            dl[1] = 0.0
        de = randn(g, N, std=0.3) if with_ent else None
        keep = x.clone()
        if inplace:
            d, ldd = x, x.stride(0)
        else:
            buf = torch.full((N, V + 5), 3.0, device=DEV, dtype=dt)
            d, ldd = buf[:, :V], V + 5
        call("ta_token_logp_bwd" + sfx, P(x), x.stride(0), P(t), F(c), P(lse),
             P(ent) if with_ent else None, P(dl), P(de), P(d), ldd, N, V, S())
        check_bwd(keep, t, c32, d, dl, de, V)
        if not inplace:  # nothing outside the rows
            assert (buf[:, V:] == 3.0).all() and torch.equal(x, keep)


def test_rows_without_token_are_not_read():
    N, V = 9, 3001
    x = torch.full((N, V), NAN, device=DEV, dtype=BF16)
    x[4] = randn(gen(1), V, dtype=BF16)
    t = torch.full((N,), -1, device=DEV, dtype=torch.int32)
    t[4] = 17
    o = [full(N) for _ in range(3)]
    call("ta_token_logp_fwd", P(x), V, P(t), F(1), *map(P, o), N, V, S())
    for v in o:
        assert torch.isfinite(v).all() and (v[:4] == 0).all() and (v[5:] == 0).all() and v[4] != 0
    g, d = full(N, NAN), torch.empty_like(x)
    g[4] = 2.0
    call("ta_token_logp_bwd", P(x), V, P(t), F(1), P(o[1]), None, P(g), None, P(d), V, N, V, S())
    assert (d[:4] == 0).all() and (d[5:] == 0).all() and torch.isfinite(d[4]).all()
    w = full(N, NAN)
    w[4] = 0.0  # masked by the weight this time
    lp, lo, kl = full(N), full(N), full(N)
    call("ta_policy_loss_logits", P(x), V, P(t), F(1), None, None, P(full(N, NAN)), P(w), F(0.2),
         F(0.2), F(0), F(0.1), F(0.5), P(lp), P(o[2]), P(lo), P(kl), P(d), V, N, V, S())
    for v in (lp, lo, kl, d, o[2]):
        assert (v == 0).all()


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("V", [40, 4099, 151936])
def test_special_logits(V, dtype):
    """-Inf in places, everywhere; +Inf; NaN; the type's lowest value; tokens
    outside the vocabulary."""
    dt, sfx = (BF16, "") if dtype == "bf16" else (torch.float32, "_f32")
    low = torch.finfo(dt).min
    g = gen(V)
    x = rows(g, 10, V, dt)
    t = torch.arange(10, device=DEV, dtype=torch.int32)
    x[0, V // 2:] = -INF                 # a masked half
    x[1, :] = -INF
    x[1, 1] = 0.25                       # one logit left, the token's
    x[2, :] = -INF                       # nothing left
    x[3, 5] = INF
    x[4, V - 1] = NAN
    x[5, :] = low                        # all at the lowest value: uniform
    x[6, :] = low
    x[6, 6] = 1.0                        # the token alone above it
    x[7, 7] = -INF                       # the token itself masked
    t[8] = V                             # no such token
    t[9] = 2 ** 31 - 1
    o = [full(10) for _ in range(3)]
    call("ta_token_logp_fwd" + sfx, P(x), V, P(t), F(1), *map(P, o), 10, V, S())
    lp, lse, ent = [v.double().cpu() for v in o]
    wl, ws, we, _ = [v.cpu() for v in ref_logp(x, torch.where(t < V, t, torch.zeros_like(t)), 1.0)]
    for r in (0, 6, 7):
        assert lp[r] == wl[r] or abs(lp[r] - wl[r]) < 1e-3, (r, lp[r], wl[r])
        assert abs(ent[r] - we[r]) < 1e-3, (r, ent[r], we[r])
    assert lp[1] == 0 and lse[1] == 0.25 and ent[1] == 0
    assert abs(lp[5] + math.log(V)) < 1e-5 and abs(ent[5] - math.log(V)) < 1e-5
    for r in (2, 3, 4):
        assert torch.isnan(torch.stack([lp[r], lse[r], ent[r]])).all(), r
    assert torch.isnan(lp[8]) and torch.isnan(lp[9])
    assert abs(lse[8] - ws[8]) < 1e-4 and abs(ent[9] - we[9]) < 1e-3
    # gradient of the rows with masked places: zeros there, finite elsewhere
    dl, d = full(10, 1.0), torch.empty_like(x)
    call("ta_token_logp_bwd" + sfx, P(x), V, P(t), F(1), P(o[1]), P(o[2]), P(dl), P(dl), P(d), V,
         10, V, S())
    assert torch.isfinite(d[0]).all() and (d[0, V // 2:] == 0).all()
    assert (d[1] == 0).all() and torch.isfinite(d[6]).all()


def test_more_rows_than_blocks():
    """Past 2^20 rows a block takes several."""
    N, V = (1 << 20) + 37, 5
    g = gen(6)
    x, t = rows(g, N, V, BF16), tokens(g, N, V, 0.2)
    o = [full(N) for _ in range(3)]
    call("ta_token_logp_fwd", P(x), V, P(t), F(1), *map(P, o), N, V, S())
    check_fwd(x, t, 1.0, *o)
    dl, d = randn(g, N), torch.empty_like(x)
    call("ta_token_logp_bwd", P(x), V, P(t), F(1), P(o[1]), None, P(dl), None, P(d), V, N, V, S())
    check_bwd(x, t, 1.0, d, dl, None, V)
    # (old_logp NULL, no KL term: dlogp = -adv * weight)
    adv, w = randn(g, N), torch.rand(N, generator=g, device=DEV)
    q = [full(N) for _ in range(4)]
    call("ta_policy_loss_logits", P(x), V, P(t), F(1), None, None, P(adv), P(w), F(0.2), F(0.2),
         F(0), F(0), F(0), *map(P, q), P(d), V, N, V, S())
    check_bwd(x, t, 1.0, d, -adv * w, None, V)


@pytest.mark.parametrize("sfx", ["", "_f32"])
def test_rows_far_apart(sfx):
    """Row offsets past 2^31 elements."""
    dt = torch.float32 if sfx else BF16
    V, ld = 1003, 2 ** 31 + 21
    buf = torch.empty(ld + V, device=DEV, dtype=dt)
    x = torch.as_strided(buf, (2, V), (ld, 1))
    x.copy_(rows(gen(3), 2, V, dt))
    keep = x.clone()
    t = torch.tensor([5, 900], device=DEV, dtype=torch.int32)
    o = [full(2) for _ in range(3)]
    call("ta_token_logp_fwd" + sfx, P(x), ld, P(t), F(1), *map(P, o), 2, V, S())
    check_fwd(keep, t, 1.0, *o)
    dl = randn(gen(4), 2)
    call("ta_token_logp_bwd" + sfx, P(x), ld, P(t), F(1), P(o[1]), None, P(dl), None, P(x), ld, 2,
         V, S())
    check_bwd(keep, t, 1.0, x, dl, None, V)


# ── LM head scoring ────────────────────────────────────────────────────────
HEADS = [(1, 1, 1), (1, 1000, 64), (3, 257, 7), (64, 128, 128), (130, 2049, 96), (65, 5000, 200),
         (300, 3001, 256), (257, 1537, 64), (1, 151936, 896), (17, 32000, 512), (512, 20000, 1536),
         (700, 40001, 128)]


@pytest.mark.parametrize("N,V,H", HEADS)
def test_lm_head_logp(N, V, H):
    g = gen(N + V + H)
    for pad, c in ((0, 1.0), (8, 0.6), (3, 1.0)):
        h = randn(g, N, H + pad, dtype=BF16)[:, :H]
        W = randn(g, V, H + pad, std=2.0 / math.sqrt(H), dtype=BF16)[:, :H]
        t = tokens(g, N, V, 0.2 if N > 8 else 0.0)
        o = [full(N) for _ in range(3)]
        call("ta_lm_head_logp", P(h), H + pad, P(W), H + pad, P(t), F(c), 0, *map(P, o), N, V, H,
             None, S())
        x = h.double() @ W.double().t()
        c32 = float(np.float32(c))
        wl, ws, we, lp = ref_logp(x, t, c32)
        # each logit is an F32 sum of H products, added at most H deep
        per = (h.double().abs() @ W.double().abs().t()).amax(1) * c32 * (H + 4) * EPS
        tol = sum_tol(V) + per * 2 + 4 * EPS * (x.abs().amax(1) * c32 * 2 + math.log(V) + 1)
        close(o[0], wl, tol, "logp")
        close(o[1], ws, tol, "lse")
        # dH = -sum p (log p + H) dx: at most 2 (log V + 1) max|dx|
        close(o[2], we, 4 * (math.log(V) + 2) * tol, "entropy")
        # the caller's workspace, without the entropy: the same bits
        ws_ = torch.empty(tadapt.lib().ta_lm_head_logp_ws(N, V, H), device=DEV, dtype=torch.uint8)
        o2 = [full(N) for _ in range(2)]
        call("ta_lm_head_logp", P(h), H + pad, P(W), H + pad, P(t), F(c), 0, *map(P, o2), None, N,
             V, H, P(ws_), S())
        assert torch.equal(o[0], o2[0]) and torch.equal(o[1], o2[1])
        # rounded logits: those of the GEMM, in another order of the sums
        lg = torch.empty(N, V, device=DEV, dtype=BF16)
        call("ta_gemm_rm", 1, 1, N, V, H, F(1), P(h), H + pad, P(W), H + pad, F(0), P(lg), V, None,
             S())
        call("ta_lm_head_logp", P(h), H + pad, P(W), H + pad, P(t), F(c), 1, *map(P, o), N, V, H,
             None, S())
        p2 = [full(N) for _ in range(3)]
        call("ta_token_logp_fwd", P(lg), V, P(t), F(c), *map(P, p2), N, V, S())
        # a logit next to a rounding border may fall on either side of it: the
        # token's by one BF16 step, the sums by p of a few such logits
        step = 2.0 ** -7 * x.abs().amax(1) * c32
        close(o[0], p2[0], step + 2 * tol, "logp, rounded")
        frac = ((o[0] - p2[0]).abs() > 0.1 * step + 2 * tol).double().mean()
        assert N < 64 or frac < 0.05, frac


@pytest.mark.parametrize("N,V,H,pad", [(257, 1501, 64, 0), (700, 1501, 192, 8),
                                       (1300, 1501, 100, 3), (9000, 1501, 64, 0),
                                       (1300, 30011, 64, 0)])  # the last in 256 x 256 tiles
@pytest.mark.parametrize("masked", [0.0, 0.4, 0.97, 1.0])
def test_lm_head_logp_masked_rows(N, V, H, pad, masked):
    """Rows without a token are left out of the product, wherever they lie;
    what the others give does not depend on them."""
    g = gen(N + H)
    h = randn(g, N, H + pad, dtype=BF16)[:, :H]
    W = randn(g, V, H, std=2.0 / math.sqrt(H), dtype=BF16)
    every = tokens(g, N, V, 0.0)
    t = torch.where(torch.rand(N, generator=g, device=DEV) < masked, torch.full_like(every, -5), every)
    if masked == 0.4:  # a prompt at the start, padding at the end, the last row alone
        t[:200] = -1
        t[N - 90:N - 1] = -1
        t[N - 1] = 7
        every[N - 1] = 7
    h.masked_fill_((t < 0)[:, None], NAN)
    want, o = [full(N) for _ in range(3)], [full(N) for _ in range(3)]
    call("ta_lm_head_logp", P(h), H + pad, P(W), H, P(every), F(1), 0, *map(P, want), N, V, H, None,
         S())
    call("ta_lm_head_logp", P(h), H + pad, P(W), H, P(t), F(1), 0, *map(P, o), N, V, H, None, S())
    on = t >= 0
    for a, b in zip(o, want):
        assert (a[~on] == 0).all() and torch.equal(a[on], b[on])


def test_lm_head_logp_infinite_inputs():
    """A NaN in one row of h stays in that row; an infinite weight gives rows
    of NaN, as the definition does."""
    N, V, H = 70, 700, 128
    g = gen(8)
    h, W = randn(g, N, H, dtype=BF16), randn(g, V, H, std=0.1, dtype=BF16)
    h[3, 5] = NAN
    t = tokens(g, N, V, 0.0)
    o = [full(N) for _ in range(3)]
    call("ta_lm_head_logp", P(h), H, P(W), H, P(t), F(1), 0, *map(P, o), N, V, H, None, S())
    for v in o:
        assert torch.isnan(v[3]) and torch.isfinite(v[:3]).all() and torch.isfinite(v[4:]).all()
    t[5] = V
    t[6] = -2
    call("ta_lm_head_logp", P(h), H, P(W), H, P(t), F(1), 0, *map(P, o), N, V, H, None, S())
    assert torch.isnan(o[0][5]) and torch.isfinite(o[1][5]) and all(v[6] == 0 for v in o)


# ── preference loss ────────────────────────────────────────────────────────
def ref_pref(logp, ref, tgt, off, kind, average, beta, sm, margin, scale):
    logp, tgt, off = logp.double().cpu(), tgt.cpu(), off.cpu().tolist()
    ref = ref.double().cpu() if ref is not None else torch.zeros_like(logp)
    N, n = len(logp), len(off) // 2
    loss, rew, d = np.zeros(n), np.zeros((n, 2)), np.full(N, np.nan)
    for p in range(n):
        idx, pi, rf = [], [], []
        for q in (2 * p, 2 * p + 1):
            b = min(max(off[q], 0), N)
            e = min(max(off[q + 1], b), N)
            d[b:e] = 0.0
            i = [j for j in range(b, e) if tgt[j] >= 0]
            k = 1.0 / len(i) if average and i else 1.0
            idx.append(i)
            pi.append(math.fsum(logp[j].item() for j in i) * k)
            rf.append(math.fsum(ref[j].item() for j in i) * k)
        rew[p] = [beta * (pi[0] - rf[0]), beta * (pi[1] - rf[1])]
        if not (idx[0] and idx[1]):
            continue
        u = (pi[0] - rf[0]) - (pi[1] - rf[1])
        z = beta * u - margin
        if kind == 0:
            loss[p] = (1 - sm) * np.logaddexp(0, -z) + sm * np.logaddexp(0, z)
            du = beta * (1 / (1 + math.exp(-max(min(z, 700), -700))) - (1 - sm))
        elif kind == 1:
            loss[p], du = (u - margin - 0.5 / beta) ** 2, 2 * (u - margin - 0.5 / beta)
        else:
            loss[p], du = max(0.0, 1 - z), -beta if z < 1 else 0.0
        for s_, i in ((1, idx[0]), (-1, idx[1])):
            for j in i:
                d[j] = s_ * scale * du * (1.0 / len(i) if average else 1.0)
    return loss, rew, d


def run_pref(logp, ref, tgt, off, kind, average, beta, sm, margin, scale, N=None):
    n = (off.numel() - 1) // 2
    loss, rew, d = full(n), torch.full((n, 2), 7.0, device=DEV), full(logp.numel(), 7.0)
    call("ta_preference_loss", P(logp), P(ref), P(tgt), P(off), n, logp.numel() if N is None else N,
         kind, average, F(beta), F(sm), F(margin), F(scale), P(loss), P(rew), P(d), S())
    return loss.cpu().numpy(), rew.cpu().numpy(), d.cpu().numpy()


def check_pref(got, want):
    """The sums are in 64 bits of F32 inputs: only the final rounding to F32
    is left (with z, u of up to 1e4 in the exponent: 1e4 2^-53), and the
    conversion of the F32 arguments."""
    for a, b, what in zip(got, want, ("loss", "rewards", "dlogp")):
        free = np.isnan(b)
        np.testing.assert_allclose(a[~free], b[~free], rtol=4 * EPS, atol=1e-30, err_msg=what)
        assert (a[free] == 7.0).all(), what


@pytest.mark.parametrize("kind", [0, 1, 2])
@pytest.mark.parametrize("lens", [[1, 1], [0, 3], [5, 0, 300, 2, 1, 1], [64, 65, 255, 256, 257, 513],
                                  [4000, 3990, 1, 9000], [20000, 30001]])
def test_preference_loss(kind, lens):
    for average in (0, 1):
        for with_ref in (True, False):
            g = gen(sum(lens) + kind * 7 + average)
            n = sum(lens)
            logp = -randn(g, n + 9).square()
            ref = logp + randn(g, n + 9, std=0.1) if with_ref else None
            tgt = tokens(g, n + 9, 50, 0.3)
            off = torch.tensor(np.cumsum([2] + lens), device=DEV, dtype=torch.int64)
            f32 = lambda v: float(np.float32(v))
            par = (kind, average, f32(0.1), f32(0.1), f32(0.05), f32(0.25))
            check_pref(run_pref(logp, ref, tgt, off, *par), ref_pref(logp, ref, tgt, off, *par))


def test_preference_masks_and_bad_offsets():
    """A sequence with no counting token, masked tokens that hold NaN, offsets
    outside 0 .. N or falling, tokens of no sequence."""
    g = gen(5)
    N = 400
    logp, ref, tgt = -randn(g, N).square(), -randn(g, N).square(), tokens(g, N, 9, 0.0)
    tgt[100:200] = -1
    logp[100:200] = NAN
    ref[150] = INF
    par = (0, 0, 0.5, 0.0, 0.0, 1.0)
    off = torch.tensor([0, 50, 100, 200, 300, 320, 390], device=DEV, dtype=torch.int64)
    got = run_pref(logp, ref, tgt, off, *par)
    check_pref(got, ref_pref(logp, ref, tgt, off, *par))
    assert got[0][1] == 0 and (got[2][100:300] == 0).all() and np.isfinite(got[0]).all()
    for bad in ([-5, 30, 10, 2000, 3000], [2 ** 62, -2 ** 62, 0, 50, 90], [10, 5, 2, 1, 0]):
        off = torch.tensor(bad, device=DEV, dtype=torch.int64)
        got = run_pref(logp, ref, tgt, off, *par)
        check_pref(got, ref_pref(logp, ref, tgt, off, *par))
    # no token at all
    off = torch.zeros(3, device=DEV, dtype=torch.int64)
    assert run_pref(logp, ref, tgt, off, *par, N=0)[0][0] == 0


def test_preference_extremes_and_optional_outputs():
    """Margins far past exp's range; NaN and Inf of counting tokens; outputs
    left out."""
    tgt = torch.zeros(4, device=DEV, dtype=torch.int32)
    off = torch.tensor([0, 1, 2, 3, 4], device=DEV, dtype=torch.int64)
    logp = torch.tensor([0.0, -5e4, -5e4, 0.0], device=DEV)
    loss, _, d = run_pref(logp, None, tgt, off, 0, 0, 1.0, 0.0, 0.0, 1.0)
    assert loss.tolist() == [0.0, 5e4] and d.tolist() == [0.0, 0.0, -1.0, 1.0]
    for kind in (0, 1, 2):
        logp[0] = NAN
        loss, rew, d = run_pref(logp, None, tgt, off, kind, 0, 1.0, 0.0, 0.0, 1.0)
        assert np.isnan(loss[0]) and np.isnan(d[:2]).all() and np.isfinite(loss[1])
    for v in (NAN, INF):
        logp[0] = v
        loss, rew, d = run_pref(logp, None, tgt, off, 1, 0, 1.0, 0.0, 0.0, 1.0)
        assert not np.isfinite(loss[0]) and loss[1] == (-5e4 - 0.5) ** 2 and not np.isfinite(d[0])
    loss = full(2)
    call("ta_preference_loss", P(logp), None, P(tgt), P(off), 2, 4, 2, 0, F(1), F(0), F(0), F(1),
         P(loss), None, None, S())
    assert loss[1] == 50001.0


def test_preference_gradient_by_differences():
    """Central differences of the loss itself: with h = 2^-6 the third
    derivative leaves h^2 / 6 (beta^3 / 10 at most for the sigmoid, 0 for the
    square) and the F32 loss 2^-24 |loss| / h."""
    g = gen(12)
    lens = [7, 5, 3, 9]
    n, h = sum(lens), 2.0 ** -6
    logp, tgt = -randn(g, n).square(), tokens(g, n, 9, 0.2)
    ref = logp + randn(g, n, std=0.3)
    off = torch.tensor(np.cumsum([0] + lens), device=DEV, dtype=torch.int64)
    for kind in (0, 1):
        par = (kind, 1, 0.5, 0.125 if kind == 0 else 0.0, 0.25, 1.0)
        loss, _, d = run_pref(logp, ref, tgt, off, *par)
        for j in range(n):
            up, dn = logp.clone(), logp.clone()
            up[j] += h
            dn[j] -= h
            step = (up[j].double() - dn[j].double()).item()
            num = (run_pref(up, ref, tgt, off, *par)[0].astype(np.float64).sum()
                   - run_pref(dn, ref, tgt, off, *par)[0].astype(np.float64).sum()) / step
            tol = h * h / 6 * 0.125 + 4 * EPS * np.abs(loss).sum() / h
            assert abs(num - d[j]) <= tol, (kind, j, num, d[j], tol)


# ── policy loss ────────────────────────────────────────────────────────────
def ref_policy(logp, old, ref, adv, w, lo, hi, dual, kb, ec=0.0, ent=None):
    lp, A, w = logp.double(), adv.double(), w.double()
    lr = lp - old.double() if old is not None else torch.zeros_like(lp)
    far = lr.abs() > 60
    r = lr.clamp(-60, 60).exp()
    pg = -torch.minimum(r * A, r.clamp(1 - lo, 1 + hi) * A)
    flat = torch.where(A >= 0, r > 1 + hi, r < 1 - lo) | far
    if dual:
        cap = (A < 0) & (r > dual)
        pg, flat = torch.where(cap, -dual * A, pg), flat | cap
    g = torch.where(flat, torch.zeros_like(r), -A * r)
    kl = torch.zeros_like(r)
    if ref is not None:
        d = ref.double() - lp
        kl = d.clamp(-60, 60).expm1() - d.clamp(-60, 60)
        g = g - kb * torch.where(d.abs() > 60, torch.zeros_like(d), d.expm1())
    loss = pg + kb * kl - (ec * ent if ent is not None else 0.0)
    on = w != 0
    z = torch.zeros_like(r)
    return torch.where(on, loss, z), torch.where(on, kl, z), torch.where(on, g * w, z)


def policy_inputs(g, N, logp, spread=0.4):
    f = dict(old=logp - randn(g, N, std=spread), ref=logp + randn(g, N, std=0.5), adv=randn(g, N))
    f["weight"] = torch.rand(N, generator=g, device=DEV) * (torch.rand(N, generator=g, device=DEV) < 0.7)
    return f


def f32(v):
    return float(np.float32(v))


@pytest.mark.parametrize("N", [1, 2, 255, 256, 257, 4099, 100003])
def test_policy_loss(N):
    g = gen(N)
    logp = -randn(g, N).square() * 3
    i = policy_inputs(g, N, logp, 0.7)
    if N > 300:
        i["old"][:20] = logp[:20] + 100.0  # a ratio of e^-100
        i["old"][20:40] = logp[20:40] - 100.0
        i["ref"][40:60] = logp[40:60] + 80.0
        i["adv"][60:80] = 0.0
    for old, ref, dual in ((True, True, 3.0), (False, True, 0.0), (True, False, 0.0),
                           (False, False, 1.5)):
        o = [full(N) for _ in range(3)]
        args = (i["old"] if old else None, i["ref"] if ref else None, i["adv"], i["weight"])
        call("ta_policy_loss", P(logp), *map(P, args), F(0.2), F(0.28), F(dual), F(0.04),
             *map(P, o), N, S())
        want = ref_policy(logp, *args, f32(0.2), f32(0.28), dual, f32(0.04))
        # everything in 64 bits from F32 inputs, rounded once (relative to the
        # loss' terms, which may cancel; results of up to e^60)
        pg = want[0] - f32(0.04) * want[1]
        close(o[0], want[0], 4 * EPS * (pg.abs() + want[1].abs()) + 1e-30, "loss")
        close(o[1], want[1], 4 * EPS * want[1].abs() + 1e-30, "kl")
        close(o[2], want[2], 4 * EPS * want[2].abs() + 1e-30, "dlogp")
    d = full(N)
    call("ta_policy_loss", P(logp), *map(P, args), F(0.2), F(0.28), F(dual), F(0.04), None, None,
         P(d), N, S())
    assert torch.equal(d, o[2])


def test_policy_loss_masked_and_nan():
    N = 300
    g = gen(2)
    logp = -randn(g, N).square()
    i = policy_inputs(g, N, logp)
    i["weight"][:100] = 0.0
    i["weight"][100:] = 0.5
    for k in ("old", "ref", "adv"):
        i[k][:50] = NAN
        i[k][50:100] = INF
    lp = logp.clone()
    lp[:100] = NAN
    i["adv"][150], i["ref"][151], i["old"][152], lp[153] = NAN, NAN, NAN, NAN
    o = [full(N) for _ in range(3)]
    call("ta_policy_loss", P(lp), P(i["old"]), P(i["ref"]), P(i["adv"]), P(i["weight"]), F(0.2),
         F(0.2), F(0), F(0.1), *map(P, o), N, S())
    for v in o:
        assert (v[:100] == 0).all()
    for v in (o[0], o[2]):
        assert torch.isnan(v[150:154]).all()
        assert torch.isfinite(v[154:]).all() and torch.isfinite(v[100:150]).all()


def test_policy_gradient_by_differences():
    """Away from the clip's edges the loss is smooth: central differences with
    h = 2^-8; |L'''| <= |A| r + kl_beta e^d, F32 rounding of the loss 2^-24 |L| / h."""
    N, h = 512, 2.0 ** -8
    g = gen(3)
    logp = -randn(g, N).square()
    i = policy_inputs(g, N, logp, 0.3)
    i["weight"] = full(N, 1.0)
    lr = (logp - i["old"]).double()
    near = ((lr - math.log(1.25)).abs() < 3 * h) | ((lr - math.log(0.75)).abs() < 3 * h)

    def run(lp):
        o = [full(N) for _ in range(3)]
        call("ta_policy_loss", P(lp), P(i["old"]), P(i["ref"]), P(i["adv"]), P(i["weight"]),
             F(0.25), F(0.25), F(0), F(0.125), *map(P, o), N, S())
        return o
    o = run(logp)
    up, dn = logp + h, logp - h
    num = (run(up)[0].double() - run(dn)[0].double()) / (up.double() - dn.double())
    third = i["adv"].double().abs() * (lr + h).exp() + 0.125 * (i["ref"] - logp + h).double().exp()
    tol = h * h / 6 * third + 4 * EPS * (o[0].double().abs() + o[1].double()) / h
    close(torch.where(near, num, o[2].double()), torch.where(near, num, num), tol + near * 1e9)


@pytest.mark.parametrize("N,V", [(1, 3), (3, 100), (40, 1000), (9, 50257), (5, 151936), (2, 170001)])
def test_policy_loss_logits(N, V):
    """The fused form against its three parts, which are checked on their own."""
    for pad, c, ec, inplace in ((0, 1.0, 0.0, False), (5, 0.8, 0.01, True), (8, 1.0, 0.02, False)):
        print(N, V, pad, c, ec, inplace, flush=True)
        g = gen(N + V + pad)
        x = rows(g, N, V, BF16, pad)
        t = tokens(g, N, V, 0.2 if N > 4 else 0.0)
        lp, lse, ent = full(N), full(N), full(N)
        call("ta_token_logp_fwd", P(x), x.stride(0), P(t), F(c), P(lp), P(lse), P(ent), N, V, S())
        i = policy_inputs(g, N, lp)
        ref = i["ref"] if pad else None
        keep = x.clone()
        d, ldd = (x, x.stride(0)) if inplace else (torch.empty(N, V, device=DEV, dtype=BF16), V)
        o = [full(N) for _ in range(4)]
        call("ta_policy_loss_logits", P(x), x.stride(0), P(t), F(c), P(i["old"]), P(ref),
             P(i["adv"]), P(i["weight"]), F(0.2), F(0.3), F(2.0), F(0.04), F(ec), P(o[0]),
             P(o[1]) if ec else None, P(o[2]), P(o[3]), P(d), ldd, N, V, S())
        w = torch.where(t >= 0, i["weight"], torch.zeros_like(i["weight"]))
        on = w != 0
        wl, _, we, _ = ref_logp(keep, torch.where(on, t, torch.full_like(t, -1)), f32(c))
        span = keep.double().abs().amax(1) * c * 2 + math.log(V) + 1
        ltol = sum_tol(V) + 4 * EPS * span
        close(o[0], wl, ltol, "logp")
        if ec:
            close(o[1], we, 4 * (math.log(V) + 2) * sum_tol(V), "entropy")
        # the loss and dlogp of the logp that came out, up to its rounding: the
        # kernel goes on with the logp before it is rounded to F32, which the
        # result is within EPS |logp| of; d(loss) = |A| r + kl_beta |1 - e^d|
        # and d(kl) = |1 - e^d| times that (r, e^d of the rounded logp, the
        # second order and far ratios within the factor 1.01)
        want = ref_policy(o[0], i["old"], ref, i["adv"], w, f32(0.2), f32(0.3), 2.0, f32(0.04),
                          f32(ec), o[1].double() if ec else None)
        off = EPS * o[0].double().abs() * 1.01
        dkl = (ref.double() - o[0]).expm1().abs() if ref is not None else 0.0
        dpg = i["adv"].double().abs() * (o[0].double() - i["old"]).exp()
        close(o[2], want[0], 8 * EPS * (want[0].abs() + want[1].abs() + f32(ec) * 13)
              + off * (dpg + f32(0.04) * dkl) + 1e-30, "loss")
        close(o[3], want[1], 8 * EPS * want[1].abs() + off * dkl + 1e-30, "kl")
        # (loss and gradient of the same call cannot be told apart further)
        check_bwd(keep, torch.where(on, t, torch.full_like(t, -1)), f32(c), d, want[2].float(),
                  (-f32(ec) * w).float() if ec else None, V)


# ── together ───────────────────────────────────────────────────────────────
def preference_chain(x, t, off, ref, V, bufs, st):
    n, N = (off.numel() - 1) // 2, x.shape[0]
    lp, lse, loss, rew, dl, d = bufs
    call("ta_token_logp_fwd", P(x), V, P(t), F(1), P(lp), P(lse), None, N, V, st)
    call("ta_preference_loss", P(lp), P(ref), P(t), P(off), n, N, 0, 0, F(0.1), F(0), F(0),
         F(1.0 / n), P(loss), P(rew), P(dl), st)
    call("ta_token_logp_bwd", P(x), V, P(t), F(1), P(lse), None, P(dl), None, P(d), V, N, V, st)


def chain_bufs(N, n, V):
    return [full(N), full(N), full(n), torch.empty(n, 2, device=DEV), full(N),
            torch.empty(N, V, device=DEV, dtype=BF16)]


def test_preference_run_from_hidden_states():
    """A preference step's losses as a program runs them: the reference's
    log-probabilities by the LM head's scoring, the policy's from its logits,
    the pairs' loss, the gradient of the logits; then once more as a captured
    graph, replayed with new contents, and on two streams at once."""
    V, H, lens = 5003, 192, [20, 31, 1, 17, 40, 25]
    N, n = sum(lens), len(lens) // 2
    g = gen(77)
    off = torch.tensor(np.cumsum([0] + lens), device=DEV, dtype=torch.int64)
    W = randn(g, V, H, std=2 / math.sqrt(H), dtype=BF16)
    h0, t = randn(g, N, H, dtype=BF16), tokens(g, N, V, 0.2)
    h1 = (h0.float() + 0.1 * randn(g, N, H)).to(BF16)
    ref, rl = full(N), full(N)
    call("ta_lm_head_logp", P(h0), H, P(W), H, P(t), F(1), 1, P(ref), P(rl), None, N, V, H, None,
         S())
    x = torch.empty(N, V, device=DEV, dtype=BF16)
    call("ta_gemm_rm", 1, 1, N, V, H, F(1), P(h1), H, P(W), H, F(0), P(x), V, None, S())
    bufs = chain_bufs(N, n, V)
    preference_chain(x, t, off, ref, V, bufs, S())
    lp, lse, loss, rew, dl, d = bufs
    check_fwd(x, t, 1.0, lp, lse, None)
    want = ref_pref(lp, ref, t, off, 0, 0, f32(0.1), 0.0, 0.0, f32(1.0 / n))
    check_pref((loss.cpu().numpy(), rew.cpu().numpy(), dl.cpu().numpy()), want)
    check_bwd(x, t, 1.0, d, dl, None, V)
    # captured
    x2 = x.clone()
    b2 = chain_bufs(N, n, V)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        preference_chain(x2, t, off, ref, V, b2, S())
    torch.cuda.synchronize()
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr, stream=st):
        preference_chain(x2, t, off, ref, V, b2, S())
    for k in range(3):
        x2.copy_(rows(gen(100 + k), N, V, BF16))
        eager = chain_bufs(N, n, V)
        preference_chain(x2, t, off, ref, V, eager, S())
        for b in b2:
            b.fill_(5.0)
        gr.replay()
        torch.cuda.synchronize()
        for a, b in zip(eager, b2):
            assert torch.equal(a, b), k
    # two streams at once
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    e1, e2 = chain_bufs(N, n, V), chain_bufs(N, n, V)
    torch.cuda.synchronize()
    for _ in range(4):
        for s, xx, e in ((s1, x, e1), (s2, x2, e2)):
            with torch.cuda.stream(s):
                preference_chain(xx, t, off, ref, V, e, S())
    torch.cuda.synchronize()
    for a, b in zip(e1, bufs):
        assert torch.equal(a, b)
    for a, b in zip(e2, eager):
        assert torch.equal(a, b)


def test_lm_head_logp_captured_twice():
    """Two graphs of one stream, each with its own workspace, replayed at the
    same time on two streams."""
    N, V, H = 130, 4000, 128
    g = gen(9)
    W = randn(g, V, H, std=2 / math.sqrt(H), dtype=BF16)
    hs = [randn(g, N, H, dtype=BF16) for _ in range(2)]
    t = tokens(g, N, V, 0.0)
    need = tadapt.lib().ta_lm_head_logp_ws(N, V, H)
    ws = [torch.empty(need, device=DEV, dtype=torch.uint8) for _ in range(2)]
    outs = [[full(N) for _ in range(3)] for _ in range(2)]
    graphs = []

    def run(k, o, w):
        call("ta_lm_head_logp", P(hs[k]), H, P(W), H, P(t), F(1), 0, *map(P, o), N, V, H, P(w), S())
    cap = torch.cuda.Stream()
    torch.cuda.synchronize()
    refused = []
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr, stream=cap):
        try:
            run(0, outs[0], None)  # the pool's buffer is not for graphs
        except tadapt.BackendError as e:
            refused.append(str(e))
        outs[0][0].fill_(1.0)
    assert refused and "workspace" in refused[0]
    for k in range(2):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr, stream=cap):
            run(k, outs[k], ws[k])
        graphs.append(gr)
    want = [[full(N) for _ in range(3)] for _ in range(2)]
    for k in range(2):
        run(k, want[k], None)
    torch.cuda.synchronize()
    st = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(3):
        for o in outs[0] + outs[1]:
            o.fill_(5.0)
        torch.cuda.synchronize()
        for k in range(2):
            with torch.cuda.stream(st[k]):
                graphs[k].replay()
        torch.cuda.synchronize()
        for k in range(2):
            for a, b in zip(outs[k], want[k]):
                assert torch.equal(a, b)


@pytest.mark.parametrize("N,V", [(3, 151936), (40, 110003)])
def test_long_rows_captured_and_eager(N, V):
    """A few long rows: eager calls split them over blocks, captured ones do
    not, so the two agree to the sums' rounding; every replay gives the same
    bits, also of another stream's graph at the same time."""
    g = gen(V)
    x, t = rows(g, N, V, BF16), tokens(g, N, V, 0.0)
    i = policy_inputs(g, N, full(N, -8.0))

    def run(o, d):
        call("ta_token_logp_fwd", P(x), V, P(t), F(1), *map(P, o[:3]), N, V, S())
        call("ta_policy_loss_logits", P(x), V, P(t), F(1), P(i["old"]), P(i["ref"]), P(i["adv"]),
             P(i["weight"]), F(0.2), F(0.3), F(0), F(0.04), F(0.01), *map(P, o[3:]), P(d), V, N, V,
             S())
    outs = [[full(N) for _ in range(7)] for _ in range(3)]
    ds = [torch.empty_like(x) for _ in range(3)]
    run(outs[0], ds[0])
    check_fwd(x, t, 1.0, *outs[0][:3])
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    graphs = []
    for k in (0, 1):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr, stream=streams[k]):
            run(outs[k + 1], ds[k + 1])
        graphs.append(gr)
    for _ in range(3):
        for o in outs[1] + outs[2] + ds[1:]:
            o.fill_(3.0)
        torch.cuda.synchronize()
        for k in (0, 1):
            with torch.cuda.stream(streams[k]):
                graphs[k].replay()
        run(outs[0], ds[0])
        torch.cuda.synchronize()
        for a, b in zip(outs[1] + [ds[1]], outs[2] + [ds[2]]):
            assert torch.equal(a, b)
        check_fwd(x, t, 1.0, *outs[1][:3])
        for k in (0, 3):
            close(outs[1][k], outs[0][k].double(), 2 * sum_tol(V) + 1e-6 * outs[0][k].abs(), "logp")
        close(ds[1], ds[0].double(), ds[0].double().abs() * 2.0 ** -6 + 1e-9, "dlogits")


def test_eager_scoring_between_replays_of_a_captured_product():
    """The scratch of scoring is not the one that a captured split-K product
    holds: growing it leaves the graph's replays right."""
    M, N, K = 64, 896, 9728
    g = gen(14)
    X, Y = randn(g, M, K, dtype=BF16), randn(g, N, K, dtype=BF16)
    C, want = torch.zeros(M, N, device=DEV, dtype=BF16), torch.zeros(M, N, device=DEV, dtype=BF16)
    st = torch.cuda.Stream()

    def product(out):
        call("ta_gemm_rm", 1, 1, M, N, K, F(1), P(X), K, P(Y), K, F(0), P(out), N, None, S())
    torch.cuda.synchronize()
    with torch.cuda.stream(st):
        product(want)
    torch.cuda.synchronize()
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr, stream=st):
        product(C)
    for V in (20000, 60000, 151936):
        h, W, t = randn(g, 300, 64, dtype=BF16), randn(g, V, 64, dtype=BF16), tokens(g, 300, V, 0.1)
        o = [full(300) for _ in range(3)]
        torch.cuda.synchronize()
        with torch.cuda.stream(st):
            call("ta_lm_head_logp", P(h), 64, P(W), 64, P(t), F(1), 0, *map(P, o), 300, V, 64, None,
                 S())
            C.zero_()
            gr.replay()
        torch.cuda.synchronize()
        assert torch.equal(C, want) and all(torch.isfinite(v).all() for v in o)
