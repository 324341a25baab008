"""The fine-tuning losses as Graph ops and as GPT training steps of the host mirror, and clipping inside the training steps.

Tolerances: the losses' own arithmetic is pinned in test_gpu_finetune.py; what the graph adds are copies and sums of fp32 values
(one rounding of 2^-24 each), and what a whole GPT adds is the matrix products' error, for which test_gpu_models.py has 1e-4 of a
tensor's scale."""
import numpy as np
import pytest

from oracle import finetune as ft
from oracle import models, ograph

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


@pytest.fixture(scope="module")
def ops():
    from znn_b200 import ops as _ops
    _ops.init(0)
    return _ops


@pytest.fixture(scope="module")
def G(ops):
    from znn_b200.graph import Graph
    return Graph


@pytest.fixture(scope="module")
def Model(ops):
    from znn_b200.models import Model as M
    return M


def relclose(a, b, tol, what, floor=0.0):
    a, b = np.asarray(a, np.float64), np.asarray(b, np.float64)
    scale = max(1e-30, float(np.abs(b).max()), floor)
    err = float(np.abs(a - b).max())
    assert err <= tol * scale, f"{what}: {err:.3e} vs scale {scale:.3e}"


def case(seed, M=37, V=130):
    r = np.random.default_rng(seed)
    x = (r.standard_normal((M, V)) * 2).astype(np.float32)
    t = r.integers(0, V, M).astype(np.int32)
    t[r.random(M) < 0.2] = -1
    used = t >= 0
    logp = ft.rows(np.where(used[:, None], x, 0), t)[0]
    old = (logp - np.log(r.choice([0.6, 0.9, 1.05, 1.6], M))).astype(np.float32)
    ref = (logp + 0.3 * r.standard_normal(M)).astype(np.float32)
    return x, t, old, r.standard_normal(M).astype(np.float32), ref


# ------------------------------------------------------------------ graph ops
def test_policy_op_is_the_entry_point(ops, G):
    x, t, old, adv, ref = case(1)
    want = ops.policy_loss(x, t, old, adv, ref, None, (0.2, 0.3), 0.1, 0.02, 0.8)
    g = G()
    X = g.array(x, True)
    loss = g.policyLoss(X, t, g.array(old), g.array(adv), g.array(ref), None, (0.2, 0.3), 0.1, 0.02, 0.8)
    assert loss.shape == (1, 2)
    np.testing.assert_array_equal(loss.data.reshape(-1), [want["loss"], want["rows"]])
    g.backward(loss)
    np.testing.assert_array_equal(X.grad, want["dlogits"])
    w = np.abs(adv)
    g2 = G()
    X2 = g2.array(x, True)
    l2 = g2.policyLoss(X2, t, g2.array(old), g2.array(adv), None, g2.array(w))
    g2.backward(l2)
    want2 = ops.policy_loss(x, t, old, adv, None, w)
    np.testing.assert_array_equal(X2.grad, want2["dlogits"])
    np.testing.assert_array_equal(l2.data.reshape(-1)[0], want2["loss"])


def test_policy_gradient_adds_to_what_is_there(ops, G):
    """Two losses on one tensor, another consumer of it, a zeroed gradient, a tape that ran again: the gradient is the sum each time."""
    x, t, old, adv, ref = case(2)
    a, b = ops.policy_loss(x, t, old, adv)["dlogits"], ops.policy_loss(x, t, old, adv, ref, None, (0.2, 0.2), 0.5)["dlogits"]
    g = G()
    X = g.array(x, True)
    l1 = g.policyLoss(X, t, g.array(old), g.array(adv))
    l2 = g.policyLoss(X, t, g.array(old), g.array(adv), g.array(ref), None, (0.2, 0.2), 0.5)
    g.backward(l1)
    np.testing.assert_array_equal(X.grad, a)
    g.backward(l2)
    np.testing.assert_array_equal(X.grad, a + b)
    g.zeroGrad()
    g.backward(l1)
    np.testing.assert_array_equal(X.grad, a)
    g.forward()
    np.testing.assert_array_equal(X.grad, a)     # the tape's forward leaves gradients alone
    g.backward(l1)
    np.testing.assert_array_equal(X.grad, a + a)
    # both losses under one sum, beside a scaled copy
    for order in (0, 1):
        g = G()
        X = g.array(x, True)
        mk = [lambda: g.policyLoss(X, t, g.array(old), g.array(adv)),
              lambda: g.policyLoss(X, t, g.array(old), g.array(adv), g.array(ref), None, (0.2, 0.2), 0.5)]
        p, q = mk[order](), mk[1 - order]()
        Y = g.mulScalar(X, 3.0)
        s = g.add(p, q)
        g.backward(s)
        np.testing.assert_allclose(X.grad, a + b, rtol=0, atol=4 * U * np.abs(a + b).max())
        Y.set_grad(np.ones_like(x))
        g.backwardWithGrad(Y)
        np.testing.assert_allclose(X.grad, a + b + 3.0, rtol=0, atol=4 * U * 4)


def test_reading_the_gradient_early_costs_nothing(ops, G):
    x, t, old, adv, _ = case(3)
    want = ops.policy_loss(x, t, old, adv)["dlogits"]
    g = G()
    X = g.array(x, True)
    loss = g.policyLoss(X, t, g.array(old), g.array(adv))
    assert np.all(X.grad == 0.0)                 # nothing has been propagated yet
    g.backward(loss)
    np.testing.assert_array_equal(X.grad, want)


def test_without_lazy_gradients(ops, G, Model):
    x, t, old, adv, _ = case(4)
    want = ops.policy_loss(x, t, old, adv)["dlogits"]
    m = Model("mlp", (4, 3, 3, 2))
    m.set_option("lazy_zero_grad", 0)
    try:
        g = G()
        X = g.array(x, True)
        loss = g.policyLoss(X, t, g.array(old), g.array(adv))
        g.backward(loss)
        np.testing.assert_array_equal(X.grad, want)
    finally:
        m.set_option("lazy_zero_grad", 1)


def test_token_logprob_and_preference_ops(ops, G):
    x, t, _, _, ref = case(5, M=24)
    off = np.array([0, 5, 11, 11, 20], np.int32)
    logp, _, stats = ops.token_logprob_fwd(x, t, 0.7, want_entropy=False)
    pref = ops.preference_loss(logp, off, ref, t, 0.4, 0.1, 0.05, True)
    want = ops.token_logprob_bwd(x, t, stats, pref["dlogp"], inv_temp=0.7)
    g = G()
    X = g.array(x, True)
    L = g.tokenLogProb(X, t, 0.7)
    assert L.shape == (24, 1)
    np.testing.assert_array_equal(L.data.reshape(-1), logp)
    loss = g.preferenceLoss(L, off, g.array(ref), t, 0.4, 0.1, 0.05, True)
    np.testing.assert_array_equal(loss.data.reshape(-1), [pref["loss"]])
    g.backward(loss)
    np.testing.assert_array_equal(L.grad.reshape(-1), pref["dlogp"])
    np.testing.assert_array_equal(X.grad, want)
    # two losses on the same log-probabilities: their gradients add, and so do two uses of the logits
    g = G()
    X = g.array(x, True)
    L = g.tokenLogProb(X, t, 0.7)
    one = g.preferenceLoss(L, off, g.array(ref), t, 0.4, 0.1, 0.05, True)
    two = g.preferenceLoss(L, off, None, None, 0.2)
    g.backward(g.add(one, two))
    p2 = ops.preference_loss(logp, off, None, None, 0.2)
    np.testing.assert_allclose(L.grad.reshape(-1), pref["dlogp"] + p2["dlogp"], rtol=0, atol=2 * U * 0.2)


def test_graph_refusals(ops, G):
    from znn_b200._lib import ZnnError
    x, t, old, adv, ref = case(6, M=8)
    g = G()
    X, o, a = g.array(x, True), g.array(old), g.array(adv)

    def refused(f, word):
        with pytest.raises(ZnnError) as e:
            f()
        assert e.value.code == -1 and word in str(e.value), e.value
    refused(lambda: g.policyLoss(X, t[:-1], o, a), "8 integers")
    refused(lambda: g.policyLoss(X, t, g.array(old[:5]), a), "one value per row")
    refused(lambda: g.policyLoss(X, t, o, a, None, None, (0.2, 0.2), 0.1), "ref_logp")
    refused(lambda: g.tokenLogProb(g.array(np.zeros((2, 3, 4), np.float32)), np.zeros(6)), "2 integers")
    refused(lambda: g.tokenLogProb(g.array(np.zeros((2, 3, 4), np.float32)), np.zeros(2)), "2-D")
    refused(lambda: g.tokenLogProb(X, t, 0.0), "inv_temp")
    L = g.tokenLogProb(X, t)
    refused(lambda: g.preferenceLoss(L, [0]), "pair")
    refused(lambda: g.preferenceLoss(L, [0, 1, 2], g.array(ref[:3])), "one value per row")
    refused(lambda: g.preferenceLoss(L, [0, 1, 2], None, t[:4]), "8 integers")


# ------------------------------------------------------------------ GPT steps
CFG = {"vocab_size": 67, "block_size": 24, "n_embd": 32, "n_head": 2, "n_layer": 2}
DIMS = (67, 24, 32, 2, 2)


def gpt(Model, seed=3):
    P = models.init_params("gpt", CFG, seed=seed)
    m = Model("gpt", DIMS, arena_bytes=256 << 20)
    m.set_params(P)
    m.set_option("lr", 0.01)
    return m, P


def tokens(seed, B=4, T=20):
    r = np.random.default_rng(seed)
    ids = r.integers(0, 67, (B, T)).astype(np.float32)
    t = np.concatenate([ids[:, 1:], r.integers(0, 67, (B, 1))], 1).astype(np.int32)
    t[:, :5] = -1          # the prompt
    t[1, 14:] = -1         # padding
    return r, ids, t


def oracle_grads(P, ids, dlogits_of):
    """The CPU restatement's parameter gradients from a gradient of the logits"""
    g = ograph.OGraph()
    T = {k: g.array(v, True) for k, v in P.items()}
    lg = models.gpt(g, T, g.array(ids, False), CFG)
    logits = g.reshape(lg, (lg.shape[0] * lg.shape[1], lg.shape[2]))
    out = dlogits_of(logits.data)
    logits.grad[...] = out["dlogits"]
    g.backwardWithGrad(logits)
    return out, {k: v.grad.reshape(P[k].shape) for k, v in T.items()}


def check_grads(got, want, what):
    floor = 0.01 * max(float(np.abs(v).max()) for v in want.values())
    for k in want:
        relclose(got[k], want[k], 1e-4, f"{what} {k}", floor)


def test_token_logprobs(Model):
    m, P = gpt(Model)
    _, ids, t = tokens(1)
    logits = m.forward(ids, seq=20, classes=67)
    lp, en = m.token_logprobs(ids, t, 0.9, want_entropy=True)
    wl, we = ft.rows(logits, t.reshape(-1), float(np.float32(0.9)))[:2]
    relclose(lp.reshape(-1), wl, 1e-6, "logp")
    relclose(en.reshape(-1), we, 1e-6, "entropy")
    assert np.all(lp[t < 0] == 0.0)
    np.testing.assert_array_equal(m.token_logprobs(ids, t, 0.9), lp)


@pytest.mark.parametrize("kl,ce,weighted", [(0.0, 0.0, False), (0.1, 0.02, True)])
def test_policy_step(Model, kl, ce, weighted):
    m, P = gpt(Model)
    r, ids, t = tokens(2)
    lp = m.token_logprobs(ids, t)
    ratio = r.choice([0.6, 0.95, 1.1, 1.5], ids.shape)
    old, ref, adv = lp - np.log(ratio).astype(np.float32), lp + 0.2 * r.standard_normal(ids.shape).astype(np.float32), r.standard_normal(ids.shape)
    old, ref, adv = (a.astype(np.float32) for a in (old, ref, adv))
    w = r.random(ids.shape).astype(np.float32) if weighted else None
    kl, ce = float(np.float32(kl)), float(np.float32(ce))
    f = lambda a: None if a is None else a.reshape(-1)   # noqa: E731
    want, grads = oracle_grads(P, ids, lambda x: ft.policy(x, f(t), f(old), f(adv), f(ref), f(w), (0.2, 0.3), kl, ce))
    loss = m.policy_step(ids, t, old, adv, ref if kl else None, w, (0.2, 0.3), kl, ce)
    assert abs(loss - want["loss"]) <= 1e-4 * max(1.0, abs(want["loss"]))
    check_grads(m.get_grads(), grads, "policy step")
    after = m.get_params()
    for k in P:
        relclose(after[k], P[k] - 0.01 * grads[k], 1e-5, k, 0.1)


def test_preference_step(Model):
    m, P = gpt(Model)
    r, ids, t = tokens(3)
    ref = (m.token_logprobs(ids, t) + 0.1 * r.standard_normal(ids.shape)).astype(np.float32)
    off = np.arange(5) * 20

    def dlogits(x):
        lp = ft.rows(x, t.reshape(-1))[0]
        p = ft.preference(lp, off, ref.reshape(-1), t.reshape(-1), float(np.float32(0.3)), float(np.float32(0.1)), 0.0, True)
        return {**p, "dlogits": ft.rows_grad(x, t.reshape(-1), p["dlogp"], np.zeros(80))}
    want, grads = oracle_grads(P, ids, dlogits)
    loss, rewards = m.preference_step(ids, t, ref, 0.3, 0.1, 0.0, True)
    assert abs(loss - want["loss"]) <= 1e-5
    np.testing.assert_allclose(rewards.reshape(-1), want["rewards"], atol=1e-5)
    check_grads(m.get_grads(), grads, "preference step")


def test_model_refusals(Model):
    from znn_b200._lib import ZnnError
    m, _ = gpt(Model)
    _, ids, t = tokens(4)
    z = np.zeros(ids.shape, np.float32)
    mlp = Model("mlp", (4, 3, 3, 2))

    def refused(f, word):
        with pytest.raises(ZnnError) as e:
            f()
        assert word in str(e.value), e.value
    refused(lambda: mlp.token_logprobs(ids, t), "not a GPT")
    refused(lambda: mlp.policy_step(ids, t, z, z), "not a GPT")
    refused(lambda: m.policy_step(ids, t, z, z, kl_coef=0.1), "ref_logp")
    refused(lambda: m.policy_step(ids[:0], t[:0], z[:0], z[:0]), "positive")
    refused(lambda: m.preference_step(ids[:0], t[:0]), "positive")
    refused(lambda: m.token_logprobs(np.zeros((1, 30), np.float32), np.zeros((1, 30))), "block_size")
    refused(lambda: m.grad_norm(), "max_grad_norm")
    refused(lambda: m.set_option("max_grad_norm", -1.0), "max_grad_norm")
    refused(lambda: m.set_option("max_grad_norm", float("nan")), "max_grad_norm")
    refused(lambda: m.set_option("max_grad_norm", 1e-60), "max_grad_norm")   # 0 in fp32


# ------------------------------------------------------------------ clipping in the training steps
def norm_of(grads):
    return np.sqrt(sum(float((g.astype(np.float64) ** 2).sum()) for g in grads.values()))


@pytest.mark.parametrize("adam", [False, True])
@pytest.mark.parametrize("momentum", [0.0, 0.9])
def test_training_with_clipped_gradients(Model, adam, momentum):
    """Step by step the parameters of the same model whose gradients a separate call clips; a bound that is never reached changes
    nothing, bit for bit."""
    from znn_b200 import ops
    P = models.init_params("mlp", (20, 16, 8, 5), seed=1)
    r = np.random.default_rng(2)

    def make(bound):
        m = Model("mlp", (20, 16, 8, 5))
        m.set_params(P)
        for k, v in (("lr", 0.05), ("momentum", momentum), ("optimizer", float(adam)), ("max_grad_norm", bound)):
            m.set_option(k, v)
        return m
    free, loose, tight = make(0.0), make(1e6), make(0.05)
    names = [k for k, *_ in free.params]
    w = {k: P[k].reshape(-1).copy() for k in names}
    v1, v2 = {k: np.zeros_like(w[k]) for k in names}, {k: np.zeros_like(w[k]) for k in names}
    for step in range(4):
        x, t = r.random((32, 20)).astype(np.float32), r.integers(0, 5, 32).astype(np.int32)
        free.train_step(x, t)
        loose.train_step(x, t)
        for k in names:
            np.testing.assert_array_equal(free.get_params()[k], loose.get_params()[k])
        tight.train_step(x, t)
        g = tight.get_grads()
        norm, factor = tight.grad_norm()
        assert abs(norm - norm_of(g)) <= 2 * U * norm and abs(factor - 0.05 / norm) <= 3 * U and factor < 1.0
        for k in names:
            gk = g[k].reshape(-1) * np.float32(factor)
            if adam:
                ops.adam_step(w[k], gk, v1[k], v2[k], 0.05, 0.9, 0.999, 1e-8, step + 1.0)
            else:
                ops.sgd_step(w[k], gk, v1[k] if momentum else None, 0.05, momentum)
            np.testing.assert_array_equal(tight.get_params()[k].reshape(-1), w[k])


def test_a_step_without_a_finite_norm_is_skipped(Model):
    m = Model("mlp", (20, 16, 8, 5))
    P = models.init_params("mlp", (20, 16, 8, 5), seed=1)
    m.set_params(P)
    m.set_option("max_grad_norm", 1.0)
    m.set_option("momentum", 0.9)
    x = np.ones((8, 20), np.float32)
    x[3, 4] = np.nan
    m.train_step(x, np.zeros(8, np.int32))
    norm, factor = m.grad_norm()
    assert not np.isfinite(norm) and factor == 0.0
    for k in P:
        np.testing.assert_array_equal(m.get_params()[k], P[k])
        assert np.all(m.get_velocities()[k] == 0.0)


def test_clipping_in_a_replayed_step(ops, Model):
    """The step captured into a CUDA graph clips by the norm of its own gradients at every replay; changing the bound captures anew."""
    from znn_b200._lib import lib
    P = models.init_params("mlp", (20, 16, 8, 5), seed=1)
    r = np.random.default_rng(7)
    xs, ts = r.random((12, 32, 20)).astype(np.float32) * 4, r.integers(0, 5, (12, 32)).astype(np.int32)
    out = []
    for replay in (0, 1):
        m = Model("mlp", (20, 16, 8, 5))
        m.set_params(P)
        for k, v in (("lr", 0.05), ("momentum", 0.9), ("max_grad_norm", 0.1), ("cuda_graph", replay)):
            m.set_option(k, v)
        xb, tb = ops.DevBuf(xs[0].nbytes), ops.DevBuf(ts[0].nbytes)
        norms = []
        for i in range(12):
            if i == 6:
                m.set_option("max_grad_norm", 0.4)
            lib().call("znn_memcpy_h2d", xb.ptr, xs[i].ctypes.data, xs[i].nbytes)
            lib().call("znn_memcpy_h2d", tb.ptr, ts[i].ctypes.data, ts[i].nbytes)
            m.train_step_device(xb.ptr, tb.ptr, 32)
            norms.append(m.grad_norm())
        assert m.graph_replays() == (10 if replay else 0)
        out.append((norms, m.get_params()))
    assert out[0][0] == out[1][0] and len(set(out[0][0])) == 12
    for k in P:
        np.testing.assert_array_equal(out[0][1][k], out[1][1][k])


def test_param_slab_clipped_step(ops):
    import ctypes as C
    from znn_b200._lib import lib
    L = lib()
    counts = (C.c_size_t * 3)(5, 1000, 33)
    h = C.c_void_p()
    L.call("znn_param_slab_create", counts, 3, C.byref(h))
    try:
        r = np.random.default_rng(1)
        w, g = {}, {}
        for i, n in enumerate((5, 1000, 33)):
            pw, pg = C.c_void_p(), C.c_void_p()
            L.call("znn_param_slab_tensor", h, i, C.byref(pw), C.byref(pg), None, None)
            w[i], g[i] = r.standard_normal(n).astype(np.float32), r.standard_normal(n).astype(np.float32)
            L.call("znn_memcpy_h2d", pw, w[i].ctypes.data, 4 * n)
            L.call("znn_memcpy_h2d", pg, g[i].ctypes.data, 4 * n)
        res = ops.DevBuf(ops.GRAD_NORM_FLOATS * 4)
        L.call("znn_param_slab_sgd_step_clipped", h, 0.1, 0.9, 0.5, 1.0, res.ptr)
        norm, factor = res.to_host((2,))
        want = ft.grad_norm([g[i] for i in range(3)], 1.0, 0.5)
        assert abs(norm - want[0]) <= 1.01 * U * want[0] and abs(factor - want[1]) <= 1.01 * U * want[1]
        for i, n in enumerate((5, 1000, 33)):
            pw = C.c_void_p()
            L.call("znn_param_slab_tensor", h, i, C.byref(pw), None, None, None)
            out, v = np.empty(n, np.float32), np.zeros(n, np.float32)
            L.call("znn_memcpy_d2h", out.ctypes.data, pw, 4 * n)
            ops.sgd_step(w[i], g[i] * np.float32(np.float32(0.5) * factor), v, 0.1, 0.9)
            np.testing.assert_array_equal(out, w[i])
    finally:
        L.call("znn_param_slab_destroy", h)
