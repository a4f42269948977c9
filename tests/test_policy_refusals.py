"""Argument checks of the preference and policy operators: every call here is
refused on the host, before anything is launched (no GPU needed)."""
import ctypes

import pytest

import tadapt

F = ctypes.c_float
X = ctypes.c_void_p(0x1000)   # stands for device memory; never read
ODD = ctypes.c_void_p(0x1001)


def refuse(msg, name, *args):
    with pytest.raises(tadapt.BackendError, match=msg):
        tadapt.call(name, *args)


FWD = dict(logits=X, ld=100, targets=X, inv_temp=F(1), logp=X, lse=X, entropy=None, N=4, V=100,
           stream=None)
BWD = dict(logits=X, ld=100, targets=X, inv_temp=F(1), lse=X, entropy=None, dlogp=X, dentropy=None,
           dlogits=ctypes.c_void_p(0x2000), ldd=100, N=4, V=100, stream=None)
HEAD = dict(h=X, ldh=64, W=X, ldw=64, targets=X, inv_temp=F(1), round_logits=0, logp=X, lse=X,
            entropy=None, N=4, V=100, H=64, ws=None, stream=None)
PREF = dict(logp=X, ref=X, targets=X, offsets=X, P=2, N=10, kind=0, average=0, beta=F(0.1),
            smoothing=F(0), margin=F(0), scale=F(1), pair_loss=X, rewards=X, dlogp=X, stream=None)
POL = dict(logp=X, old=X, ref=X, adv=X, weight=X, lo=F(0.2), hi=F(0.2), dual=F(0), kl_beta=F(0),
           loss=X, kl=X, dlogp=X, N=10, stream=None)
PLOG = dict(logits=X, ld=100, targets=X, inv_temp=F(1), old=X, ref=X, adv=X, weight=X, lo=F(0.2),
            hi=F(0.2), dual=F(0), kl_beta=F(0), ent_coef=F(0), logp=X, entropy=None, loss=X, kl=X,
            dlogits=ctypes.c_void_p(0x2000), ldd=100, N=4, V=100, stream=None)
INF, NAN = float("inf"), float("nan")

CASES = [
    ("ta_token_logp_fwd", FWD, [
        (dict(N=-1), "bad shape"), (dict(V=0), "bad shape"), (dict(ld=99), "bad shape"),
        (dict(V=2 ** 30 + 1, ld=2 ** 31), "bad shape"), (dict(inv_temp=F(0)), "inv_temp"), (dict(inv_temp=F(INF)), "inv_temp"),
        (dict(inv_temp=F(NAN)), "inv_temp"), (dict(logits=None), "null"),
        (dict(targets=None), "null"), (dict(logp=None), "null"), (dict(lse=None), "null"),
        (dict(logits=ODD), "misaligned")]),
    ("ta_token_logp_fwd_f32", FWD, [(dict(logits=ctypes.c_void_p(0x1002)), "misaligned")]),
    ("ta_token_logp_bwd", BWD, [
        (dict(ldd=99), "bad shape"), (dict(ld=1), "bad shape"), (dict(inv_temp=F(-1)), "inv_temp"),
        (dict(dlogp=None), "null"), (dict(lse=None), "null"), (dict(dentropy=X), "entropy"),
        (dict(dlogits=ODD), "misaligned"), (dict(dlogits=X, ldd=104), "in place")]),
    ("ta_lm_head_logp", HEAD, [
        (dict(H=0), "bad shape"), (dict(ldh=63), "bad shape"), (dict(ldw=63), "bad shape"),
        (dict(V=0), "bad shape"), (dict(inv_temp=F(0)), "inv_temp"),
        (dict(round_logits=2), "round_logits"), (dict(h=None), "null"), (dict(h=ODD), "misaligned"),
        (dict(ws=ctypes.c_void_p(0x1008)), "misaligned"), (dict(N=2 ** 31 - 1), "more tiles"),
        (dict(V=2 ** 30 + 1), "more tiles"), (dict(N=2 ** 25 + 1, V=1), "more tiles")]),
    ("ta_preference_loss", PREF, [
        (dict(P=-1), "bad shape"), (dict(N=-1), "bad shape"), (dict(kind=3), "kind"),
        (dict(average=2), "average"), (dict(beta=F(0)), "beta"), (dict(beta=F(NAN)), "beta"),
        (dict(smoothing=F(1)), "smoothing"), (dict(smoothing=F(-0.1), kind=1), "smoothing"),
        (dict(margin=F(INF)), "finite"), (dict(scale=F(NAN)), "finite"),
        (dict(offsets=None), "null"), (dict(logp=None), "null"), (dict(pair_loss=None), "null")]),
    ("ta_policy_loss", POL, [
        (dict(N=-1), "bad shape"), (dict(logp=None), "null"), (dict(adv=None), "null"),
        (dict(weight=None), "null"), (dict(dlogp=None), "null"), (dict(lo=F(1)), "clip range"),
        (dict(hi=F(-0.1)), "clip range"), (dict(hi=F(NAN)), "clip range"),
        (dict(dual=F(1)), "dual_clip"), (dict(dual=F(-2)), "dual_clip"),
        (dict(kl_beta=F(INF)), "finite")]),
    ("ta_policy_loss_logits", PLOG, [
        (dict(V=0), "bad shape"), (dict(ldd=10), "bad shape"), (dict(inv_temp=F(0)), "inv_temp"),
        (dict(ent_coef=F(0.1)), "entropy"), (dict(ent_coef=F(NAN)), "finite"),
        (dict(loss=None), "null"), (dict(weight=None), "null"), (dict(dlogits=ODD), "misaligned"),
        (dict(dlogits=X, ldd=104), "in place")]),
]


@pytest.mark.parametrize("name,good,change,msg", [
    (name, good, change, msg) for name, good, bads in CASES for change, msg in bads])
def test_refused(name, good, change, msg):
    refuse(msg, name, *dict(good, **change).values())


@pytest.mark.parametrize("name,good,empty", [
    ("ta_token_logp_fwd", FWD, dict(N=0)), ("ta_token_logp_fwd_f32", FWD, dict(N=0)),
    ("ta_token_logp_bwd", BWD, dict(N=0)), ("ta_lm_head_logp", HEAD, dict(N=0)),
    ("ta_preference_loss", PREF, dict(P=0)), ("ta_policy_loss", POL, dict(N=0)),
    ("ta_policy_loss_logits", PLOG, dict(N=0))])
def test_nothing_to_do(name, good, empty):
    """No rows: no launch, no use of the pointers."""
    args = dict(good, **empty)
    args = {k: None if isinstance(v, ctypes.c_void_p) else v for k, v in args.items()}
    assert tadapt.call(name, *args.values()) == 0


def test_workspace_size():
    L = tadapt.lib()
    assert L.ta_lm_head_logp_ws(0, 100, 64) == 0
    small, large = L.ta_lm_head_logp_ws(5, 129, 64), L.ta_lm_head_logp_ws(300, 129, 64)
    assert small >= (2 * 3 + 1) * 5 * 4 and small % 256 == 0
    assert large >= (2 * 3 + 1) * 300 * 4 + 300 * 64 * 2 + 2 * 300 * 4
