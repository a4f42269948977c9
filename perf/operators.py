"""The operators of preference and policy fine-tuning, as cases that can be timed.

An adapter that the cross entropy has trained is tuned further on pairs of
answers (a preference loss) or on its own rated answers (a clipped policy
loss).  Both are made of the log-probability of each token:

  token_logp       logits -> log-probability of each row's token, entropy;
                   and their gradient to the logits
  lm_head_logp     the same from the LM head's input and weight, the logits
                   never stored (scoring by the frozen base or an old policy)
  preference_loss  token log-probabilities of pairs of packed sequences ->
                   loss of each pair, rewards, gradient of each token
  policy_loss      token log-probabilities -> clipped policy loss with a KL
                   term, gradient of each token; or straight from the logits
                   to their gradient

  own               False: run computes plain torch; True: the framework's calls
  listed()          the named cases
  draw(rng)         one more case of the same ranges
  prepare(c, seed)  what the program holds before the call
  run(state)        one pass, and its outputs
  work(c)           bytes and flops the pass cannot do without
  exact(c, seed)    the same outputs from the definitions in 64 bits
"""
import ctypes
import math
import os
import random
import sys

import torch

own = False

DEV = "cuda"
BF16 = torch.bfloat16
# loss kinds as the framework numbers them
KINDS = {"sigmoid": 0, "ipo": 1, "hinge": 2}


def listed():
    return [
        # one token scored over the whole vocabulary: latency counts
        dict(name="logp_one_token", kind="logp", N=1, V=151936, dtype="bf16", pad=0, prompt=0.0,
             entropy=False, grad=False, inv_temp=1.0),
        # a batch of answers scored with their entropy; the prompts' rows have
        # no token
        dict(name="logp_score", kind="logp", N=4096, V=151936, dtype="bf16", pad=0, prompt=0.4,
             entropy=True, grad=False, inv_temp=1.0),
        # log-probability and entropy of a training batch at a sampling
        # temperature, and the gradient of both
        dict(name="logp_train", kind="logp", N=2048, V=152064, dtype="bf16", pad=0, prompt=0.25,
             entropy=True, grad=True, inv_temp=1.25),
        # F32 logits of a ragged batch and a vocabulary that is no multiple of
        # anything, in rows of a padded buffer
        dict(name="logp_f32_odd", kind="logp", N=777, V=50257, dtype="f32", pad=47, prompt=0.3,
             entropy=False, grad=True, inv_temp=1.0),
        # one short answer scored by the 0.5B base's LM head
        dict(name="head_short", kind="head", N=128, H=896, V=151936, prompt=0.0, entropy=False,
             inv_temp=1.0),
        # the reference log-probabilities of 8 x 1024 tokens of the 1.5B base
        dict(name="head_batch", kind="head", N=8192, H=1536, V=151936, prompt=0.0, entropy=True,
             inv_temp=1.0),
        # four pairs of short answers: latency counts
        dict(name="pref_small", kind="pref", P=4, T=300, loss="sigmoid", average=False, ref=True,
             prompt=0.3, smoothing=0.0),
        # a large batch of long pairs of packed sequences, means of the tokens
        dict(name="pref_long", kind="pref", P=32, T=4096, loss="ipo", average=True, ref=True,
             prompt=0.3, smoothing=0.0),
        # the whole way of a preference step, logits to their gradient: log-
        # probabilities, the pairs' loss, the gradient
        dict(name="pref_step", kind="pref_step", P=4, T=512, V=151936, loss="sigmoid",
             average=False, ref=True, prompt=0.3, smoothing=0.1),
        # the policy loss of a batch whose log-probabilities are at hand
        dict(name="policy_tokens", kind="policy", N=65536, prompt=0.3, ref=True, dual_clip=3.0),
        # a policy step from the logits to their gradient, with KL term and
        # entropy bonus
        dict(name="policy_step", kind="policy_step", N=2048, V=151936, prompt=0.25, ref=True,
             ent_coef=0.01, dual_clip=0.0, inv_temp=1.0),
        # the same without reference or entropy, over an odd vocabulary
        dict(name="policy_step_odd", kind="policy_step", N=500, V=50257, prompt=0.2, ref=False,
             ent_coef=0.0, dual_clip=3.0, inv_temp=1.0),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _vocab(rng):
    """Vocabulary sizes: the framework's own, other common ones, odd ones."""
    return rng.choice([151936, 152064, 32000, 50257, _log(rng, 1000, 152064)])


def draw(rng):
    kind = rng.choice(["logp", "logp", "head", "pref", "pref_step", "policy", "policy_step"])
    prompt = round(rng.uniform(0.0, 0.6), 3)
    ent = rng.random() < 0.5
    if kind == "logp":
        return dict(kind=kind, N=_log(rng, 1, 2048), V=_vocab(rng),
                    dtype=rng.choice(["bf16", "bf16", "f32"]),
                    pad=rng.choice([0, 0, 8 * rng.randint(1, 64), rng.randint(1, 100)]),
                    prompt=prompt, entropy=ent, grad=rng.random() < 0.6,
                    inv_temp=rng.choice([1.0, round(rng.uniform(0.5, 2.0), 3)]))
    if kind == "head":
        return dict(kind=kind, N=_log(rng, 1, 4096), H=64 * _log(rng, 4, 56), V=_vocab(rng),
                    prompt=prompt, entropy=ent,
                    inv_temp=rng.choice([1.0, round(rng.uniform(0.5, 2.0), 3)]))
    loss = rng.choice(sorted(KINDS))
    pair = dict(loss=loss, average=loss == "ipo" or rng.random() < 0.4, ref=rng.random() < 0.7,
                prompt=prompt, smoothing=rng.choice([0.0, 0.1]))
    if kind == "pref":
        P = _log(rng, 1, 64)
        return dict(kind=kind, P=P, T=_log(rng, 1, max(2, min(16384, 131072 // P))), **pair)
    if kind == "pref_step":
        P = _log(rng, 1, 16)
        return dict(kind=kind, P=P, T=_log(rng, 2, max(3, 2048 // P)), V=_vocab(rng), **pair)
    pol = dict(prompt=prompt, ref=rng.random() < 0.7, dual_clip=rng.choice([0.0, 3.0]))
    if kind == "policy":
        return dict(kind=kind, N=_log(rng, 1, 65536), **pol)
    return dict(kind=kind, N=_log(rng, 1, 2048), V=_vocab(rng), ent_coef=0.01 if ent else 0.0,
                inv_temp=rng.choice([1.0, round(rng.uniform(0.5, 2.0), 3)]), **pol)


# ── inputs ─────────────────────────────────────────────────────────────────
BETA, CLIP_LO, CLIP_HI, KL_BETA = 0.1, 0.2, 0.28, 0.04


class Gen:
    """Seeded tensors on the GPU."""

    def __init__(self, seed):
        self.g = torch.Generator(device=DEV)
        self.g.manual_seed(int(seed) * 1000003 + 29)

    def f32(self, *shape, std=1.0, mean=0.0):
        return torch.randn(*shape, generator=self.g, device=DEV) * std + mean

    def ints(self, hi, n):
        return torch.randint(0, hi, (n,), generator=self.g, device=DEV, dtype=torch.int32)

    def targets(self, N, V, prompt):
        """Token ids, -1 for a share of the rows in runs of up to 64 (prompts)."""
        t, n = self.ints(V, N), max(1, min(64, N // 8))
        off = torch.rand((N + n - 1) // n, generator=self.g, device=DEV) < prompt
        return torch.where(off.repeat_interleave(n)[:N], torch.full_like(t, -1), t)


def _logits(g, N, V, dtype, pad, targets):
    """Logits as a trained model gives them: spread over the vocabulary, the
    row's token among the likely ones; rows of a buffer V + pad wide."""
    buf = torch.empty(N, V + pad, device=DEV, dtype=BF16 if dtype == "bf16" else torch.float32)
    for r in range(0, N, 256):
        n = min(256, N - r)
        x = g.f32(n, V + pad, std=2.0)
        t = targets[r:r + n].clamp(min=0).long()[:, None]
        x.scatter_add_(1, t, g.f32(n, 1, std=3.0, mean=9.0))
        buf[r:r + n] = x.to(buf.dtype)
    return buf[:, :V]


def _row_logp(logits, targets, c):
    """log-probabilities in F32, as an earlier pass left them (old policy)."""
    out = torch.empty(targets.shape[0], device=DEV)
    for r in range(0, out.shape[0], 256):
        x = logits[r:r + 256].float() * c
        t = targets[r:r + 256].clamp(min=0).long()[:, None]
        out[r:r + 256] = x.gather(1, t)[:, 0] - x.logsumexp(1)
    return out


def _policy_inputs(g, s, logp, case):
    """Old and reference log-probabilities, advantages and token weights of
    rated answers.  Ratios keep clear of the clip's edges, where a last bit
    decides between a gradient and none."""
    N = logp.shape[0]
    lr = g.f32(N, std=0.15)
    for edge in (math.log(1 - CLIP_LO), math.log(1 + CLIP_HI)):
        lr = torch.where((lr - edge).abs() < 1e-3, lr + 4e-3, lr)
    s["old"] = logp - lr
    s["ref"] = logp + g.f32(N, std=0.3) if case["ref"] else None
    s["adv"] = g.f32(N)
    live = s["targets"] >= 0
    s["weight"] = live.float() / live.sum().clamp(min=1)


def _lengths(case):
    """Lengths of the 2 P sequences, 1 to T tokens."""
    rng = random.Random(case["P"] * 7919 + case["T"])
    return [rng.randint((case["T"] + 1) // 2, case["T"]) for _ in range(2 * case["P"])]


def _pair_inputs(g, s, case):
    n = _lengths(case)
    s["offsets"] = torch.tensor([sum(n[:i]) for i in range(len(n) + 1)], dtype=torch.int64,
                                device=DEV)
    return sum(n)


def prepare(case, seed):
    g, kind, s = Gen(seed), case["kind"], dict(case=case)
    f32 = dict(device=DEV, dtype=torch.float32)
    if kind == "head":
        N, H, V = case["N"], case["H"], case["V"]
        s["targets"] = g.targets(N, V, case["prompt"])
        s["W"] = torch.empty(V, H, device=DEV, dtype=BF16)
        for r in range(0, V, 16384):
            n = min(16384, V - r)
            s["W"][r:r + n] = g.f32(n, H, std=2.0 / math.sqrt(H)).to(BF16)
        s["h"] = (g.f32(N, H) + 2.0 * s["W"][s["targets"].clamp(min=0).long()].float()).to(BF16)
        outs = N
    elif kind == "pref":
        outs = _pair_inputs(g, s, case)
        s["targets"] = g.targets(outs, 1000, case["prompt"])
        s["logp"] = torch.where(s["targets"] >= 0, -g.f32(outs).square(), torch.zeros(outs, **f32))
        s["ref"] = s["logp"] + g.f32(outs, std=0.2) if case["ref"] else None
    elif kind == "policy":
        outs = case["N"]
        s["targets"] = g.targets(outs, 1000, case["prompt"])
        s["logp"] = torch.where(s["targets"] >= 0, -g.f32(outs).square(), torch.zeros(outs, **f32))
        _policy_inputs(g, s, s["logp"], case)
    else:
        outs = _pair_inputs(g, s, case) if kind == "pref_step" else case["N"]
        V, dtype, pad = case["V"], case.get("dtype", "bf16"), case.get("pad", 0)
        s["targets"] = g.targets(outs, V, case["prompt"])
        s["logits"] = _logits(g, outs, V, dtype, pad, s["targets"])
        if kind == "logp" and case["grad"]:
            s["dlogp"] = g.f32(outs)
            s["dent"] = g.f32(outs, std=0.1) if case["entropy"] else None
        if kind == "pref_step":
            # a policy that has begun to move: chosen tokens above the
            # reference, rejected ones below it
            side = torch.bucketize(torch.arange(outs, device=DEV), s["offsets"][1:], right=True) % 2
            s["ref"] = (_row_logp(s["logits"], s["targets"], 1.0) + g.f32(outs, std=0.2)
                        + 0.2 * side - 0.1 if case["ref"] else None)
        if kind == "policy_step":
            _policy_inputs(g, s, _row_logp(s["logits"], s["targets"], case["inv_temp"]), case)
        if kind != "logp" or case["grad"]:
            s["dlogits"] = torch.empty(outs, V, device=DEV, dtype=s["logits"].dtype)
    # the program's output buffers
    for k in ("o_logp", "o_lse", "o_ent", "o_loss", "o_kl", "o_dlogp"):
        s[k] = torch.empty(outs, **f32)
    if "P" in case:
        s["o_pair"] = torch.empty(case["P"], **f32)
        s["o_rew"] = torch.empty(case["P"], 2, **f32)
    return s


# ── the plain forms ────────────────────────────────────────────────────────
def _plain_logp(logits, targets, c, entropy):
    """(logp, lse, entropy, p log p parts) of F32 logits; masked rows 0."""
    live = targets >= 0
    x = logits.float() * c
    m = x.amax(1, keepdim=True)
    e = torch.exp(x - m)
    # in 64 bits: a sequence adds up the errors of hundreds of rows
    lsum = torch.log(e.sum(1, keepdim=True, dtype=torch.float64))
    lse = (m + lsum).float()
    xt = x.gather(1, targets.clamp(min=0).long()[:, None])
    zero = torch.zeros_like(lse[:, 0])
    logp = torch.where(live, ((xt - m) - lsum).float()[:, 0], zero)
    ent = None
    if entropy:
        d = (e * torch.where(e > 0, x - m, torch.zeros_like(x))).sum(1, keepdim=True)
        ent = torch.where(live, (lsum - d / torch.exp(lsum)).float()[:, 0], zero)
    return logp, torch.where(live, lse[:, 0], zero), ent


def _plain_dlogits(logits, targets, c, lse, ent, g, e):
    live = (targets >= 0)[:, None]
    lp = logits.float() * c - lse[:, None]
    p = torch.exp(lp)
    d = -g[:, None] * p
    d.scatter_add_(1, targets.clamp(min=0).long()[:, None], g[:, None])
    if e is not None:
        d = d - e[:, None] * p * (lp + ent[:, None])
    return torch.where(live, d * c, torch.zeros_like(d)).to(logits.dtype)


def _plain_pref(s, case, logp):
    off, P = s["offsets"], case["P"]
    n = logp.shape[0]
    seq = torch.bucketize(torch.arange(n, device=DEV), off[1:], right=True)
    live = s["targets"] >= 0
    zero = torch.zeros(2 * P, dtype=torch.float64, device=DEV)

    def sums(v):
        return zero.index_add(0, seq, torch.where(live, v.double(), torch.zeros_like(v).double()))

    cnt = sums(torch.ones_like(logp))
    pi = sums(logp)
    rf = sums(s["ref"]) if s["ref"] is not None else zero
    if case["average"]:
        pi, rf = pi / cnt.clamp(min=1), rf / cnt.clamp(min=1)
    u = (pi[0::2] - pi[1::2]) - (rf[0::2] - rf[1::2])
    z, sm = BETA * u, case["smoothing"]
    if case["loss"] == "sigmoid":
        sp = torch.clamp(z, min=0) + torch.log1p(torch.exp(-z.abs()))  # softplus(z)
        loss = (1 - sm) * (sp - z) + sm * sp
        du = BETA * (torch.sigmoid(z) - (1 - sm))
    elif case["loss"] == "ipo":
        q = u - 1 / (2 * BETA)
        loss, du = q * q, 2 * q
    else:
        loss = torch.clamp(1 - z, min=0)
        du = torch.where(z < 1, torch.full_like(z, -BETA), torch.zeros_like(z))
    both = (cnt[0::2] > 0) & (cnt[1::2] > 0)
    loss = torch.where(both, loss, torch.zeros_like(loss))
    du = torch.where(both, du, torch.zeros_like(du)) / P
    dseq = torch.stack([du, -du], 1).reshape(-1)
    if case["average"]:
        dseq = dseq / cnt.clamp(min=1)
    dlogp = torch.where(live, dseq[seq], torch.zeros_like(dseq[seq])).float()
    rew = (BETA * (pi - rf)).reshape(P, 2).float()
    return loss.float(), rew, dlogp


def _plain_policy(s, case, logp, ent):
    live = s["weight"] != 0
    zero = torch.zeros_like(logp)
    lp, A = logp.double(), s["adv"].double()
    r = torch.exp(lp - s["old"].double())
    pg = -torch.minimum(r * A, torch.clamp(r, 1 - CLIP_LO, 1 + CLIP_HI) * A)
    flat = torch.where(A >= 0, r > 1 + CLIP_HI, r < 1 - CLIP_LO)
    if case["dual_clip"]:
        cap = -case["dual_clip"] * A
        flat = flat | ((A < 0) & (pg > cap))
        pg = torch.where(A < 0, torch.minimum(pg, cap), pg)
    g = torch.where(flat, torch.zeros_like(pg), -A * r)
    kl = torch.zeros_like(pg)
    if s["ref"] is not None:
        d = s["ref"].double() - lp
        kl = torch.expm1(d) - d
        g = g - KL_BETA * torch.expm1(d)
    loss = pg + KL_BETA * kl
    if ent is not None:
        loss = loss - case["ent_coef"] * ent.double()
    return (torch.where(live, loss.float(), zero), torch.where(live, kl.float(), zero),
            torch.where(live, (g * s["weight"]).float(), zero))


def _run_plain(s):
    case = s["case"]
    kind, c = case["kind"], case.get("inv_temp", 1.0)
    if kind in ("logp", "head"):
        x = s["logits"] if kind == "logp" else s["h"].float() @ s["W"].float().t()
        logp, lse, ent = _plain_logp(x, s["targets"], c, case["entropy"])
        out = dict(logp=logp, lse=lse)
        if case["entropy"]:
            out["entropy"] = ent
        if case.get("grad"):
            out["dlogits"] = _plain_dlogits(x, s["targets"], c, lse, ent, s["dlogp"], s["dent"])
        return out
    if kind == "pref":
        loss, rew, dlogp = _plain_pref(s, case, s["logp"])
        return dict(loss=loss, rewards=rew, dlogp=dlogp)
    if kind == "policy":
        loss, kl, dlogp = _plain_policy(s, case, s["logp"], None)
        return dict(loss=loss, kl=kl, dlogp=dlogp)
    ec = case.get("ent_coef", 0.0)
    logp, lse, ent = _plain_logp(s["logits"], s["targets"], c, ec != 0)
    if kind == "pref_step":
        loss, rew, dlogp = _plain_pref(s, case, logp)
        out = dict(logp=logp, loss=loss, rewards=rew)
    else:
        loss, kl, dlogp = _plain_policy(s, case, logp, ent)
        out = dict(logp=logp, loss=loss, kl=kl)
        if ec:
            out["entropy"] = ent
    out["dlogits"] = _plain_dlogits(s["logits"], s["targets"], c, lse, ent, dlogp,
                                    -ec * s["weight"] if ec else None)
    return out


# ── the framework's calls ──────────────────────────────────────────────────
def _run_own(s):
    path = os.path.join(os.getcwd(), "tensor-adapt_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import tadapt
    P, call, st = tadapt.ptr, tadapt.call, tadapt.stream()
    F = ctypes.c_float
    case = s["case"]
    kind, c = case["kind"], F(case.get("inv_temp", 1.0))
    tgt = P(s["targets"])
    if "logits" in s:
        x = s["logits"]
        N, V, ld = x.shape[0], x.shape[1], x.stride(0)
        sfx = "" if x.dtype == BF16 else "_f32"
    if kind == "logp":
        ent = s["o_ent"] if case["entropy"] else None
        call("ta_token_logp_fwd" + sfx, P(x), ld, tgt, c, P(s["o_logp"]), P(s["o_lse"]), P(ent),
             N, V, st)
        out = dict(logp=s["o_logp"], lse=s["o_lse"])
        if ent is not None:
            out["entropy"] = ent
        if case["grad"]:
            call("ta_token_logp_bwd" + sfx, P(x), ld, tgt, c, P(s["o_lse"]), P(ent),
                 P(s["dlogp"]), P(s["dent"]), P(s["dlogits"]), V, N, V, st)
            out["dlogits"] = s["dlogits"]
        return out
    if kind == "head":
        ent = s["o_ent"] if case["entropy"] else None
        call("ta_lm_head_logp", P(s["h"]), case["H"], P(s["W"]), case["H"], tgt, c, 0,
             P(s["o_logp"]), P(s["o_lse"]), P(ent), case["N"], case["V"], case["H"], None, st)
        out = dict(logp=s["o_logp"], lse=s["o_lse"])
        if ent is not None:
            out["entropy"] = ent
        return out
    if kind == "policy":
        call("ta_policy_loss", P(s["logp"]), P(s["old"]), P(s["ref"]), P(s["adv"]),
             P(s["weight"]), F(CLIP_LO), F(CLIP_HI), F(case["dual_clip"]), F(KL_BETA),
             P(s["o_loss"]), P(s["o_kl"]), P(s["o_dlogp"]), case["N"], st)
        return dict(loss=s["o_loss"], kl=s["o_kl"], dlogp=s["o_dlogp"])
    if kind == "policy_step":
        ent = s["o_ent"] if case["ent_coef"] else None
        call("ta_policy_loss_logits", P(x), ld, tgt, c, P(s["old"]), P(s["ref"]), P(s["adv"]),
             P(s["weight"]), F(CLIP_LO), F(CLIP_HI), F(case["dual_clip"]), F(KL_BETA),
             F(case["ent_coef"]), P(s["o_logp"]), P(ent), P(s["o_loss"]), P(s["o_kl"]),
             P(s["dlogits"]), V, N, V, st)
        out = dict(logp=s["o_logp"], loss=s["o_loss"], kl=s["o_kl"])
        if ent is not None:
            out["entropy"] = ent
        out["dlogits"] = s["dlogits"]
        return out
    logp = s.get("logp")
    if kind == "pref_step":
        logp = s["o_logp"]
        call("ta_token_logp_fwd", P(x), ld, tgt, c, P(logp), P(s["o_lse"]), None, N, V, st)
    call("ta_preference_loss", P(logp), P(s["ref"]), tgt, P(s["offsets"]), case["P"],
         logp.shape[0], KINDS[case["loss"]], int(case["average"]), F(BETA), F(case["smoothing"]),
         F(0.0), F(1.0 / case["P"]), P(s["o_pair"]), P(s["o_rew"]), P(s["o_dlogp"]), st)
    if kind == "pref":
        return dict(loss=s["o_pair"], rewards=s["o_rew"], dlogp=s["o_dlogp"])
    call("ta_token_logp_bwd", P(x), ld, tgt, c, P(s["o_lse"]), None, P(s["o_dlogp"]), None,
         P(s["dlogits"]), V, N, V, st)
    return dict(logp=logp, loss=s["o_pair"], rewards=s["o_rew"], dlogits=s["dlogits"])


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ── what a pass cannot do without ──────────────────────────────────────────
def _live_rows(case, N):
    """Rows with a token, in the mean over the seeds: a run of rows is a
    prompt with the probability case["prompt"]."""
    return N * (1.0 - case["prompt"])


def work(case):
    kind = case["kind"]
    if kind == "head":
        N, H, V = _live_rows(case, case["N"]), case["H"], case["V"]
        return dict(bytes=2.0 * (N * H + V * H) + 16.0 * case["N"], flops=2.0 * N * V * H)
    if kind == "policy":
        return dict(bytes=case["N"] * (28.0 + (4.0 if case["ref"] else 0.0)), flops=30.0 * case["N"])
    if "P" in case:
        n = sum(_lengths(case))
        small = n * (12.0 + (4.0 if case["ref"] else 0.0))
        if kind == "pref":
            return dict(bytes=small, flops=8.0 * n)
    n = n if "P" in case else case["N"]
    live, V = _live_rows(case, n), case["V"]
    es = 4.0 if case.get("dtype") == "f32" else 2.0
    grad = kind != "logp" or case["grad"]
    # each logit read once, each gradient written once (masked rows' too)
    return dict(bytes=es * V * (live + (n if grad else 0)) + 24.0 * n,
                flops=(12.0 if grad else 5.0) * live * V)


# ── the definitions in 64 bits ─────────────────────────────────────────────
def _exact_rows(x, tgt, c):
    """float64 log-softmax of scaled rows: (log p, lse)."""
    x = x * c
    m = x.max(1, keepdim=True).values
    lse = m + (x - m).exp().sum(1, keepdim=True).log()
    return x - lse, lse[:, 0]


def _exact_pairs(s, case, logp):
    """Pair by pair, in Python floats."""
    off = s["offsets"].tolist()
    live = (s["targets"] >= 0).cpu()
    lp = logp.double().cpu()
    rf = s["ref"].double().cpu() if s["ref"] is not None else torch.zeros_like(lp)
    loss, rew, dlp = [], [], torch.zeros_like(lp)
    sm = case["smoothing"]
    for p in range(case["P"]):
        tot, refs, cnt, idx = [], [], [], []
        for q in (2 * p, 2 * p + 1):
            i = torch.nonzero(live[off[q]:off[q + 1]])[:, 0] + off[q]
            k = float(len(i)) if case["average"] and len(i) else 1.0
            idx.append(i), cnt.append(len(i))
            tot.append(math.fsum(lp[i].tolist()) / k), refs.append(math.fsum(rf[i].tolist()) / k)
        u = (tot[0] - refs[0]) - (tot[1] - refs[1])
        z = BETA * u
        if case["loss"] == "sigmoid":
            neg = math.log1p(math.exp(-abs(z))) + max(-z, 0.0)  # -log sigma(z)
            pos = math.log1p(math.exp(-abs(z))) + max(z, 0.0)
            sg = 1 / (1 + math.exp(-z)) if z >= 0 else math.exp(z) / (1 + math.exp(z))
            L, du = (1 - sm) * neg + sm * pos, BETA * (sm * sg - (1 - sm) * (1 - sg))
        elif case["loss"] == "ipo":
            L, du = (u - 0.5 / BETA) ** 2, 2 * (u - 0.5 / BETA)
        else:
            L, du = max(0.0, 1 - z), -BETA if z < 1 else 0.0
        if not (cnt[0] and cnt[1]):
            L, du = 0.0, 0.0
        for q, sign in ((0, 1.0), (1, -1.0)):
            if cnt[q]:
                dlp[idx[q]] = sign * du / case["P"] / (cnt[q] if case["average"] else 1)
        loss.append(L), rew.append([BETA * (tot[0] - refs[0]), BETA * (tot[1] - refs[1])])
    f64 = dict(dtype=torch.float64, device=DEV)
    return torch.tensor(loss, **f64), torch.tensor(rew, **f64).reshape(-1, 2), dlp.to(DEV)


def _exact_policy(s, case, logp, ent):
    live = s["weight"] != 0
    A, lp = s["adv"].double(), logp.double()
    lr = lp - s["old"].double()
    hi, lo = math.log1p(CLIP_HI), math.log1p(-CLIP_LO)
    # the objective is r A inside the clip's edge on A's side, flat outside
    edge = torch.where(A >= 0, lr.clamp(max=hi), lr.clamp(min=lo))
    slope = (edge == lr).double()
    if case["dual_clip"]:
        top = math.log(case["dual_clip"])
        slope = torch.where((A < 0) & (lr > top), torch.zeros_like(slope), slope)
        edge = torch.where(A < 0, edge.clamp(max=top), edge)
    loss, g = -A * edge.exp(), -A * lr.exp() * slope
    kl = torch.zeros_like(loss)
    if s["ref"] is not None:
        d = s["ref"].double() - lp
        kl = d.expm1() - d
        loss, g = loss + KL_BETA * kl, g - KL_BETA * d.expm1()
    if ent is not None:
        loss = loss - case["ent_coef"] * ent
    return loss * live, kl * live, g * s["weight"].double()


def exact(case, seed):
    s, kind, c = prepare(case, seed), case["kind"], case.get("inv_temp", 1.0)
    if kind == "pref":
        return dict(zip(("loss", "rewards", "dlogp"), _exact_pairs(s, case, s["logp"])))
    if kind == "policy":
        return dict(zip(("loss", "kl", "dlogp"), _exact_policy(s, case, s["logp"], None)))
    tgt, f64 = s["targets"], dict(dtype=torch.float64, device=DEV)
    N = tgt.shape[0]
    logp, lse, ent = (torch.zeros(N, **f64) for _ in range(3))
    w64 = s["W"].double().t() if kind == "head" else None

    def rows(r, n):
        x = s["h"][r:r + n].double() @ w64 if kind == "head" else s["logits"][r:r + n].double()
        return _exact_rows(x, tgt, c)

    step = 256
    for r in range(0, N, step):
        lp, ls = rows(r, step)
        on = (tgt[r:r + step] >= 0).double()
        t = tgt[r:r + step].clamp(min=0).long()[:, None]
        logp[r:r + step] = lp.gather(1, t)[:, 0] * on
        lse[r:r + step] = ls * on
        ent[r:r + step] = -(lp.exp() * lp).sum(1) * on
    out = dict(logp=logp)
    use_ent = case.get("entropy") or case.get("ent_coef")
    if kind in ("logp", "head"):
        out["lse"] = lse
        g, e = s.get("dlogp"), s.get("dent")
    elif kind == "pref_step":
        out["loss"], out["rewards"], g = _exact_pairs(s, case, logp)
        e = None
    else:
        out["loss"], out["kl"], g = _exact_policy(s, case, logp, ent if use_ent else None)
        e = -case["ent_coef"] * s["weight"] if use_ent else None
    if use_ent:
        out["entropy"] = ent
    if "dlogits" not in s:
        return out
    d = torch.zeros(N, case["V"], **f64)
    for r in range(0, N, step):
        lp, _ = rows(r, step)
        p, t = lp.exp(), tgt[r:r + step].long()[:, None]
        gr = g[r:r + step, None].double()
        one = torch.arange(case["V"], device=DEV)[None] == t
        x = gr * (one.double() - p)
        if e is not None:
            x = x - e[r:r + step, None].double() * p * (lp + ent[r:r + step, None])
        d[r:r + step] = x * c * (t >= 0)
    out["dlogits"] = d
    return out
