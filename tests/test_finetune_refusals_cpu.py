"""Argument checks of the fine-tuning operators: refused before anything reaches a device, so they run anywhere."""
import ctypes as C

import pytest

from znn_b200 import _lib

INVALID = -1
P = 4096   # stands for a device pointer: no refused call looks at what it points to


@pytest.fixture(scope="module")
def L():
    import os
    if not os.path.exists(_lib.LIB_PATH):
        from znn_b200 import build
        build.build()
    return _lib.lib()


def refused(L, name, *args):
    with pytest.raises(_lib.ZnnError) as e:
        L.call(name, *args)
    assert e.value.code == INVALID, e.value
    return str(e.value)


FWD = dict(logits=P, ld=8, targets=P, inv_temp=1.0, logp=P, entropy=P, stats=P, M=4, N=8)


@pytest.mark.parametrize("change,word", [(dict(logits=None), "NULL"), (dict(targets=None), "NULL"), (dict(logp=None), "NULL"), (dict(ld=7), "ld"),
                                         (dict(M=-1), "M"), (dict(N=0), "N"), (dict(inv_temp=0.0), "inv_temp"), (dict(inv_temp=-1.0), "inv_temp"),
                                         (dict(inv_temp=float("nan")), "inv_temp"), (dict(inv_temp=float("inf")), "inv_temp"),
                                         (dict(inv_temp=3e38), "inv_temp"), (dict(logits=P + 2), "aligned")])
def test_token_logprob_fwd(L, change, word):
    assert word in refused(L, "znn_token_logprob_fwd", *{**FWD, **change}.values())


BWD = dict(logits=P, ld=8, targets=P, inv_temp=1.0, stats=P, entropy=P, dlogp=P, dentropy=P, dlogits=2 * P, ld_d=8, accumulate=0, M=4, N=8)


@pytest.mark.parametrize("change,word", [(dict(logits=None), "NULL"), (dict(stats=None), "NULL"), (dict(dlogits=None), "NULL"), (dict(ld_d=7), "ld_d"),
                                         (dict(entropy=None), "entropy"), (dict(dlogits=P, accumulate=1), "own buffer"),
                                         (dict(dlogits=P, ld_d=9), "own buffer"), (dict(M=-2), "M"), (dict(dlogits=P + 3), "aligned")])
def test_token_logprob_bwd(L, change, word):
    assert word in refused(L, "znn_token_logprob_bwd", *{**BWD, **change}.values())


POLICY = dict(logits=P, ld=8, targets=P, inv_temp=1.0, old=P, ref=P, adv=P, weights=None, lo=0.2, hi=0.2, kl=0.1, ent=0.0, loss=P, token_loss=P,
              logp=P, entropy=P, dlogits=2 * P, ld_d=8, M=4, N=8)


@pytest.mark.parametrize("change,word", [(dict(old=None), "NULL"), (dict(adv=None), "NULL"), (dict(loss=None), "NULL"), (dict(token_loss=None), "NULL"),
                                         (dict(ref=None), "ref_logp"), (dict(lo=-0.1), "clip"), (dict(lo=1.5), "clip"), (dict(hi=-0.1), "clip"),
                                         (dict(hi=float("inf")), "clip"), (dict(lo=float("nan")), "clip"), (dict(kl=float("nan")), "finite"),
                                         (dict(ent=float("inf")), "finite"), (dict(ld_d=7), "ld_d"), (dict(dlogits=P, ld_d=9), "own buffer"),
                                         (dict(M=0), "M"), (dict(N=-3), "N"), (dict(ld=2), "ld"), (dict(dlogits=P + 1), "aligned"),
                                         (dict(logits=P + 1), "aligned")])
def test_policy_loss(L, change, word):
    assert word in refused(L, "znn_policy_loss", *{**POLICY, **change}.values())


PREF = dict(logp=P, ref=None, targets=None, offsets=P, beta=0.1, smooth=0.0, margin=0.0, norm=0, loss=P, pair=P, rewards=P, dlogp=P, pairs=2, M=9)


@pytest.mark.parametrize("change,word", [(dict(logp=None), "NULL"), (dict(offsets=None), "NULL"), (dict(loss=None), "NULL"), (dict(pair=None), "NULL"),
                                         (dict(rewards=None), "NULL"), (dict(pairs=0), "P"), (dict(pairs=1 << 30), "P"), (dict(M=-1), "M"),
                                         (dict(beta=float("nan")), "beta"), (dict(margin=float("inf")), "margin"), (dict(smooth=1.0), "label_smoothing"),
                                         (dict(smooth=-0.1), "label_smoothing"), (dict(smooth=float("nan")), "label_smoothing")])
def test_preference_loss(L, change, word):
    assert word in refused(L, "znn_preference_loss", *{**PREF, **change}.values())


def table(*pairs):
    n = len(pairs)
    return (C.c_void_p * n)(*[p for p, _ in pairs]), (C.c_size_t * n)(*[c for _, c in pairs]), n


def test_gradient_set(L):
    g, c, n = table((P, 4), (P, 8))
    assert "max_norm" in refused(L, "znn_grad_norm", g, c, n, 1.0, 0.0, P)
    assert "max_norm" in refused(L, "znn_grad_norm", g, c, n, 1.0, float("nan"), P)
    assert "grad_scale" in refused(L, "znn_grad_norm", g, c, n, float("nan"), 1.0, P)
    assert "result" in refused(L, "znn_grad_norm", g, c, n, 1.0, 1.0, None)
    assert "result" in refused(L, "znn_grad_norm", g, c, n, 1.0, 1.0, P + 4)
    assert "n is negative" in refused(L, "znn_grad_norm", g, c, -1, 1.0, 1.0, P)
    assert "NULL" in refused(L, "znn_grad_norm", None, c, n, 1.0, 1.0, P)
    assert "NULL" in refused(L, "znn_clip_grads", g, None, n, P)
    assert "result" in refused(L, "znn_clip_grads", g, c, n, None)
    for spans in (((P, 4), (P, 4)), ((P, 9), (P + 64, 2), (P + 32, 5)), ((P, 5), (P + 16, 1))):
        assert "overlap" in refused(L, "znn_clip_grads", *table(*spans), P)
    for bad, word in (((None, 3), "NULL"), ((P + 2, 3), "aligned"), ((P, 1 << 41), "implausible")):
        g, c, n = table((P, 4), bad)
        for name, tail in (("znn_grad_norm", (1.0, 1.0, P)), ("znn_clip_grads", (P,))):
            text = refused(L, name, g, c, n, *tail)
            assert word in text and "tensor 1" in text


def test_clipped_steps(L):
    for bad in range(3):
        ptrs = [P, P, P]
        ptrs[bad] = None
        w, g, r = ptrs
        refused(L, "znn_sgd_step_clipped", w, g, None, 0.1, 0.0, 1.0, r, 5)
        refused(L, "znn_adam_step_clipped", w, g, P, P, 0.1, 0.9, 0.99, 1e-8, 1.0, 1.0, r, 5)
    assert "velocity" in refused(L, "znn_sgd_step_clipped", P, P, None, 0.1, 0.9, 1.0, P, 5)
    assert "step count" in refused(L, "znn_adam_step_clipped", P, P, P, P, 0.1, 0.9, 0.99, 1e-8, 0.0, 1.0, P, 5)
    refused(L, "znn_adam_step_clipped", P, P, None, P, 0.1, 0.9, 0.99, 1e-8, 1.0, 1.0, P, 5)
    assert L.call("znn_sgd_step_clipped", None, None, None, 0.1, 0.0, 1.0, None, 0) == 0   # nothing to do


def test_arrays_of_the_wrong_size():
    """The numpy front end: a shorter array is refused before anything is uploaded."""
    import numpy as np
    from znn_b200 import ops
    x, t, v, short = np.zeros((4, 7), np.float32), np.zeros(4, np.int32), np.zeros(4, np.float32), np.zeros(3, np.float32)
    bad = [lambda: ops.token_logprob_fwd(x, t[:3]), lambda: ops.token_logprob_fwd(v, t), lambda: ops.token_logprob_bwd(x, t, np.zeros((3, 2)), v),
           lambda: ops.token_logprob_bwd(x, t, np.zeros((4, 2)), short), lambda: ops.token_logprob_bwd(x, t, np.zeros((4, 2)), v, dlogits=x[:3].copy()),
           lambda: ops.policy_loss(x, t, short, v), lambda: ops.policy_loss(x, t, v, short), lambda: ops.policy_loss(x, t, v, v, short),
           lambda: ops.policy_loss(x, t, v, v, None, short), lambda: ops.preference_loss(v, [0, 2]), lambda: ops.preference_loss(v, [0, 2, 4], short),
           lambda: ops.preference_loss(v, [0, 2, 4], None, t[:2]), lambda: ops.preference_loss(v, [0, 2, 4], dlogp=short),
           lambda: ops.sgd_step_clipped(v, short, None, 0.1, 0.0, 1.0), lambda: ops.adam_step_clipped(v, v, short, v, 0.1, 0.9, 0.9, 1e-8, 1.0, 1.0)]
    for f in bad:
        with pytest.raises(ValueError):
            f()


def test_values_that_are_no_32_bit_integers():
    """The numpy front end: targets and offsets are refused, not wrapped around to other tokens and rows."""
    import numpy as np
    from znn_b200 import ops
    x, v = np.zeros((4, 7), np.float32), np.zeros(4, np.float32)
    for bad in ([0, 1, 2, 2 ** 32 + 1], [0, 1, 2, -2 ** 31 - 1], [0, 1, 2, 2.5], [0, 1, 2, np.nan], [0, 1, 2, np.inf]):
        for f in (lambda: ops.token_logprob_fwd(x, np.array(bad)), lambda: ops.token_logprob_bwd(x, np.array(bad), np.zeros((4, 2)), v),
                  lambda: ops.policy_loss(x, np.array(bad), v, v), lambda: ops.preference_loss(v, [0, 2, 4], None, np.array(bad)),
                  lambda: ops.preference_loss(v, np.array([0, 2, 2 ** 32 + 4]))):
            with pytest.raises(ValueError, match="32-bit"):
                f()
    np.testing.assert_array_equal(ops.int32_array("t", np.array([[1, -2 ** 31], [2 ** 31 - 1, -7]])), np.array([[1, -2 ** 31], [2 ** 31 - 1, -7]], np.int32))
    np.testing.assert_array_equal(ops.int32_array("t", [1.0, -3.0]), np.array([1, -3], np.int32))


def test_arrays_that_cannot_be_written_in_place():
    """The numpy front end copies a result's bytes over such an array: another type, a view with gaps or a read-only one is refused."""
    import numpy as np
    from znn_b200 import ops
    v, x, t, st = np.zeros(4, np.float32), np.zeros((4, 6), np.float32), np.zeros(4, np.int32), np.zeros((4, 2), np.float32)
    fixed = v.copy()
    fixed.flags.writeable = False
    for bad in (np.zeros(4), np.zeros(8, np.float32)[::2], np.zeros(4, np.float16), fixed, [0.0] * 4):
        for f in (lambda: ops.clip_grads([v, bad], 1.0), lambda: ops.sgd_step_clipped(bad, v, None, 0.1, 0.0, 1.0),
                  lambda: ops.sgd_step_clipped(v, v, bad, 0.1, 0.9, 1.0), lambda: ops.adam_step_clipped(bad, v, v, v, 0.1, 0.9, 0.9, 1e-8, 1.0, 1.0),
                  lambda: ops.adam_step_clipped(v, v, bad, v, 0.1, 0.9, 0.9, 1e-8, 1.0, 1.0), lambda: ops.adam_step_clipped(v, v, v, bad, 0.1, 0.9, 0.9, 1e-8, 1.0, 1.0)):
            with pytest.raises(ValueError, match="in place"):
                f()
    for bad in (np.zeros((4, 6)), np.zeros((6, 4), np.float32).T, np.zeros((4, 12), np.float32)[:, ::2]):
        with pytest.raises(ValueError, match="in place"):
            ops.token_logprob_bwd(x, t, st, v, dlogits=bad)
