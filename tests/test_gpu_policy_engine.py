"""Preference and policy steps of the step engine, and its scoring.

The losses and their kernels are checked on their own in test_gpu_policy.py,
and the step's backward and AdamW against the oracle in test_gpu_step.py; here
the pieces are checked as the engine joins them: scoring against the logits in
64 bits from the engine's own final hidden states, the gradient of the logits
that a step leaves against the loss' formulas, the adapter's gradient against
differences of the loss, the update against AdamW of that gradient."""
import math

import numpy as np
import pytest
import torch

import oracle as O
import tadapt
from step_util import base_tensors, pairs
from test_gpu_policy import EPS, close, f32, ref_logp, ref_policy, ref_pref, sum_tol

pytestmark = pytest.mark.gpu

MODEL = dict(vocab=2048, hidden=256, layers=2, n_q=4, n_kv=2, head_dim=64, inter=512,
             rms_eps=1e-6, rope_theta=1e6, tie=1)
ADAPT = dict(rank=16, alpha=32.0, inject_mask=0b1111111, lr=1e-3, grad_clip=1e3, warmup=0,
             total_steps=10, b1=0.9, b2=0.999, eps=1e-8, wd=0.01)
DEV = "cuda"



def engine(B, T, seed, adapter=True, **kw):
    """An engine on a seeded base whose adapter has trained: B not zero."""
    eng = tadapt.Engine(MODEL, ADAPT, B, T, **kw)
    tensors = base_tensors(MODEL, seed)
    for name, arr in tensors.items():
        eng.set_weight(name, arr)
    rng = np.random.default_rng(seed + 1)
    if adapter:
        for l, t in pairs(MODEL, ADAPT):
            b = (rng.standard_normal(eng.adapter(l, t, "B").shape) * 0.05).astype(np.float32)
            eng.write_adapter(l, t, "B", b)
            eng.write_adapter(l, t, "B16", O.bf16_from_f32(b))
    return eng, tensors["model.embed_tokens.weight"]


def batch(B, T, seed, masked=0.3):
    rng = np.random.default_rng(seed)
    toks = rng.integers(0, MODEL["vocab"], (B, T + 1)).astype(np.int32)
    tgt = toks[:, 1:].copy()
    tgt[rng.random((B, T)) < masked] = -1
    return toks[:, :-1].reshape(-1).copy(), tgt.reshape(-1)


def logits_of(eng, W):
    """BF16-rounded logits (as the engine rounds them) from its final hidden
    states, in 64 bits."""
    x = torch.from_numpy(eng.read_buffer("xfn").view(np.int16)).view(torch.bfloat16)
    w = torch.from_numpy(np.ascontiguousarray(W).view(np.int16)).view(torch.bfloat16)
    x = x.reshape(-1, MODEL["hidden"]).double().to(DEV)
    return x @ w.reshape(-1, MODEL["hidden"]).double().to(DEV).t()


def dev(a, dt=torch.float32):
    return torch.from_numpy(np.ascontiguousarray(a)).to(DEV, dt)


@pytest.mark.parametrize("B,T", [(1, 1), (2, 33), (4, 128)])
def test_scoring(B, T):
    eng, W = engine(B, T, 3)
    plain, _ = engine(B, T, 3, adapter=False)
    inp, tgt = batch(B, T, 5, 0.3 if T > 1 else 0.0)
    t = dev(tgt, torch.int32)
    for use in (True, False):
        logp, ent = eng.logp(inp, tgt, use_adapter=use, entropy=True)
        x = logits_of(eng, W)
        lg = x.float().bfloat16()
        wl, _, we, _ = ref_logp(lg, t, 1.0)
        # a logit next to a rounding border may fall on its other side: one
        # BF16 step of it, 2^-8 of its size on either side
        tol = 2.0 ** -7 * x.abs().amax(1) + sum_tol(MODEL["vocab"]) * 4
        close(dev(logp), wl, tol, "logp")
        close(dev(ent), we, 4 * (math.log(MODEL["vocab"]) + 2) * tol, "entropy")
        assert (logp[tgt < 0] == 0).all() and (ent[tgt < 0] == 0).all()
        if use:
            with_adapter = logp
        else:  # the base alone: an engine whose adapter adds nothing
            np.testing.assert_allclose(logp, plain.logp(inp, tgt), atol=float(tol.max()))
            assert np.abs(logp - with_adapter).max() > 10 * float(tol.max())
    # scoring changes no state
    m = eng.step(inp, tgt)
    assert m["step"] == 1
    for e in (eng, plain):
        e.close()


def state_of(eng):
    return {(l, t, w): eng.adapter(l, t, w).copy() for l, t in pairs(MODEL, ADAPT)
            for w in ("A", "B", "mA", "mB", "vA", "vB")}


def check_update(eng, before, m):
    """AdamW of the gradient the step left (the rule of ops.cu:1139-1158)."""
    lr, b1, b2, eps, wd = m["lr"], ADAPT["b1"], ADAPT["b2"], ADAPT["eps"], ADAPT["wd"]
    t = m["step"]
    for l, tg in pairs(MODEL, ADAPT):
        for w in "AB":
            g = eng.adapter(l, tg, "g" + w).astype(np.float64)
            assert np.isfinite(g).all() and np.any(g), (l, tg, w)
            mm = b1 * before[l, tg, "m" + w] + (1 - b1) * g
            vv = b2 * before[l, tg, "v" + w] + (1 - b2) * g * g
            p = before[l, tg, w].astype(np.float64)
            want = p - lr * (mm / (1 - b1 ** t) / (np.sqrt(vv / (1 - b2 ** t)) + eps) + wd * p)
            np.testing.assert_allclose(eng.adapter(l, tg, w), want, rtol=1e-5, atol=1e-3 * lr)


@pytest.mark.parametrize("recompute", [False, True])
@pytest.mark.parametrize("loss,average", [("sigmoid", False), ("ipo", True), ("hinge", False)])
def test_preference_step(loss, average, recompute):
    B, T = 4, 96
    eng, W = engine(B, T, 11, recompute=recompute)
    inp, tgt = batch(B, T, 13)
    ref = eng.logp(inp, tgt, use_adapter=False)
    before = state_of(eng)
    m = eng.step_preference(inp, tgt, ref, loss=loss, average=average, beta=0.1)
    t = dev(tgt, torch.int32)
    off = torch.arange(B + 1, device=DEV) * T
    logp = eng.read_buffer("logp")
    x = logits_of(eng, W)
    wl, _, _, _ = ref_logp(x.float().bfloat16(), t, 1.0)
    close(dev(logp), wl, 2.0 ** -7 * x.abs().amax(1) + sum_tol(2048) * 4, "logp")
    want = ref_pref(dev(logp), dev(ref), t, off, tadapt.PREFERENCE_LOSSES[loss], int(average),
                    f32(0.1), 0.0, 0.0, f32(2.0 / B))
    np.testing.assert_allclose(eng.read_buffer("pair_loss"), want[0], rtol=4 * EPS)
    np.testing.assert_allclose(eng.read_buffer("rewards").reshape(-1, 2), want[1], rtol=4 * EPS)
    np.testing.assert_allclose(eng.read_buffer("dlogp"), want[2], rtol=4 * EPS, atol=1e-30)
    assert abs(m["loss"] - want[0].mean()) <= 4 * EPS * np.abs(want[0]).sum()
    assert m["valid_tokens"] == (tgt >= 0).sum() and m["nonfinite_logits"] == -1 and m["step"] == 1
    # the gradient the LM head's backward took: of logits that may differ by
    # one BF16 step, so p by 2^-7 |x|
    d = torch.from_numpy(eng.read_buffer("logits").view(np.int16)).view(torch.bfloat16)
    d = d.reshape(B * T, -1).to(DEV)
    g = dev(want[2].astype(np.float32)).double()[:, None]
    p = torch.softmax(x, 1)
    one = torch.zeros_like(p).scatter_(1, t.clamp(min=0).long()[:, None], 1.0)
    w = g * (one - p)
    close(d, w, w.abs() * 2.0 ** -8 + g.abs() * p * 2.0 ** -7 * 2 * x.abs().amax(1, keepdim=True)
          + 1e-30, "dlogits")
    check_update(eng, before, m)
    # the cross entropy step after it is a cross entropy step
    m2 = eng.step(inp, tgt)
    assert m2["step"] == 2 and abs(m2["loss"] - math.log(2048)) < 1.0
    eng.close()


def test_preference_step_starts_at_log_two():
    """Policy = reference: every margin is 0 up to the rounding borders of the
    two ways to the logits."""
    B, T = 2, 64
    eng, _ = engine(B, T, 17, adapter=False)
    inp, tgt = batch(B, T, 19, 0.0)
    ref = eng.logp(inp, tgt, use_adapter=False)
    m = eng.step_preference(inp, tgt, ref)
    assert abs(m["loss"] - math.log(2)) < 0.01 and np.abs(eng.read_buffer("rewards")).max() < 0.02
    eng.close()


@pytest.mark.parametrize("full", [False, True])
def test_policy_step(full):
    B, T = 3, 77
    eng, W = engine(B, T, 23)
    inp, tgt = batch(B, T, 29)
    rng = np.random.default_rng(31)
    N = B * T
    adv = rng.standard_normal(N).astype(np.float32)
    weight = ((tgt >= 0) * (rng.random(N) < 0.9) / max(1, (tgt >= 0).sum())).astype(np.float32)
    kw = dict(clip_lo=0.2, clip_hi=0.3)
    if full:
        old = eng.logp(inp, tgt) + (0.2 * rng.standard_normal(N)).astype(np.float32)
        ref = eng.logp(inp, tgt, use_adapter=False)
        kw.update(old_logp=old, ref_logp=ref, dual_clip=2.0, kl_beta=0.05, ent_coef=0.01)
    before = state_of(eng)
    m = eng.step_policy(inp, tgt, adv, weight, **kw)
    t, lp = dev(tgt, torch.int32), dev(eng.read_buffer("logp"))
    ent = dev(eng.read_buffer("entropy")).double()
    w = dev(weight)
    want = ref_policy(lp, dev(old) if full else None, dev(ref) if full else None, dev(adv), w,
                      f32(0.2), f32(0.3), 2.0 if full else 0.0, f32(0.05) if full else 0.0,
                      f32(0.01) if full else 0.0, ent)
    # (the loss goes on from the logp before its rounding, within EPS |logp|;
    # ratios e^1 and |A| of 5 at most here)
    slack = EPS * lp.double().abs() * 20
    close(dev(eng.read_buffer("loss_tok")), want[0], 8 * EPS * (want[0].abs() + 1) + slack, "loss")
    close(dev(eng.read_buffer("kl")), want[1], 8 * EPS * want[1].abs() + slack, "kl")
    total = float((want[0] * w.double()).sum())
    assert abs(m["loss"] - total) <= 1e-5 * float((want[0].abs() * w.double()).sum())
    assert m["valid_tokens"] == ((tgt >= 0) & (weight != 0)).sum()
    x = logits_of(eng, W)
    d = torch.from_numpy(eng.read_buffer("logits").view(np.int16)).view(torch.bfloat16)
    d = d.reshape(N, -1).to(DEV)
    live = (t >= 0) & (w != 0)
    p = torch.softmax(x, 1)
    lpx = torch.log_softmax(x, 1)
    H = -(p * lpx).sum(1, keepdim=True)
    one = torch.zeros_like(p).scatter_(1, t.clamp(min=0).long()[:, None], 1.0)
    g = want[2][:, None]
    e = (-f32(0.01) if full else 0.0) * w.double()[:, None]
    wd = torch.where(live[:, None], g * (one - p) - e * p * (lpx + H), torch.zeros_like(p))
    step = 2.0 ** -7 * x.abs().amax(1, keepdim=True)  # one BF16 step of a logit
    size = p * (g.abs() + e.abs() * (lpx.abs() + H + 1))
    close(d, wd, wd.abs() * 2.0 ** -8 + size * 4 * step + 1e-30, "dlogits")
    check_update(eng, before, m)
    eng.close()


def test_adapter_gradient_by_differences():
    """The loss at adapters moved along the gradient both ways.  The losses of
    the policy step are summed in 64 bits here from scored log-probabilities;
    what the BF16 logits leave is noise of about 2^-9 |x| = 0.01 a token, which
    the mean over 250 tokens and |A| brings below 2e-3 and the distance chosen
    (a change of the loss of about 0.2) below 2%.  One central difference s(h)
    is off by h^2 / 6 of the third derivative and terms of h^4, and
    (4 s(h / 2) - s(h)) / 3 has no h^2 left.  (The loss is that curved here: s
    is 0.97, 1.09, 1.12, 1.13 at h, h / 2, h / 4, h / 8, the norm 1.14.)"""
    B, T = 2, 125
    eng, _ = engine(B, T, 37)
    inp, tgt = batch(B, T, 41, 0.0)
    rng = np.random.default_rng(43)
    N = B * T
    adv = rng.standard_normal(N).astype(np.float32)
    weight = np.full(N, 1.0 / N, np.float32)
    old = eng.logp(inp, tgt)
    keep = {k: v for k, v in state_of(eng).items() if k[2] in "AB"}
    eng.step_policy(inp, tgt, adv, weight, old_logp=old, clip_lo=0.99, clip_hi=50.0)
    grad = {(l, t, w): eng.adapter(l, t, "g" + w) for l, t, w in keep}
    norm = math.sqrt(sum(float((g.astype(np.float64) ** 2).sum()) for g in grad.values()))
    # a direction of unit length: the loss falls norm per unit along it
    def loss_at(h):
        for (l, t, w), v in keep.items():
            p = (v + h * grad[l, t, w] / norm).astype(np.float32)
            eng.write_adapter(l, t, w, p)
            eng.write_adapter(l, t, w + "16", O.bf16_from_f32(p))
        lp = eng.logp(inp, tgt).astype(np.float64)
        return float((-np.exp(lp - old) * adv).sum() / N)
    h = 0.1 / norm
    s1 = (loss_at(h) - loss_at(-h)) / (2 * h)
    s2 = (loss_at(h / 2) - loss_at(-h / 2)) / h
    slope = (4 * s2 - s1) / 3
    print("norm", norm, "slope", slope, flush=True)
    assert abs(slope - norm) <= 0.1 * norm, (slope, norm)
    eng.close()


def test_refusals():
    eng, _ = engine(3, 8, 47)
    inp, tgt = batch(3, 8, 53)
    one = np.ones(24, np.float32)
    with pytest.raises(tadapt.BackendError, match="pairs"):
        eng.step_preference(inp, tgt)
    bad = inp.copy()
    bad[5] = 2048
    for f in (lambda i, t: eng.logp(i, t), lambda i, t: eng.step_policy(i, t, one, one)):
        with pytest.raises(tadapt.BackendError, match="token id 2048"):
            f(bad, tgt)
        with pytest.raises(tadapt.BackendError, match="target id 2048"):
            f(inp, bad)
    for kw, msg in ((dict(clip_lo=1.0), "clip range"), (dict(dual_clip=0.5), "dual_clip"),
                    (dict(inv_temp=0.0), "inv_temp"), (dict(kl_beta=float("nan")), "finite")):
        with pytest.raises(tadapt.BackendError, match=msg):
            eng.step_policy(inp, tgt, one, one, **kw)
    with pytest.raises(tadapt.BackendError, match="values for"):
        eng.logp(inp[:5], tgt)
    eng.close()
    eng, _ = engine(2, 8, 47)
    with pytest.raises(tadapt.BackendError, match="beta"):
        eng.step_preference(*batch(2, 8, 1), beta=0.0)
    # nothing was applied
    assert eng.step(*batch(2, 8, 1))["step"] == 1
    eng.close()
