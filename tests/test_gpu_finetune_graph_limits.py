"""Graph ops of the fine-tuning losses over many passes of one tape, and what a refused op leaves behind."""
import numpy as np
import pytest

from test_gpu_finetune_models import U, case

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    from znn_b200 import ops as _ops
    _ops.init(0)
    return _ops


@pytest.fixture(scope="module")
def G(ops):
    from znn_b200.graph import Graph
    return Graph


@pytest.mark.parametrize("two", [False, True])
def test_a_tape_that_runs_many_times_needs_no_more_memory(ops, G, two):
    """zeroGrad, forward, backward of one tape, hundreds of times, in an arena that has room for each loss's spare gradient once
    (logits and their gradient, two spare gradients: 4 x 19240 bytes; what is left of 160 KB holds less than another five)."""
    x, t, old, adv, ref = case(11)
    want = ops.policy_loss(x, t, old, adv)["dlogits"]
    g = G(160 << 10)
    X = g.array(x, True)
    loss = g.policyLoss(X, t, g.array(old), g.array(adv))
    if two:
        want = want + ops.policy_loss(x, t, old, adv, ref, None, (0.2, 0.2), 0.5)["dlogits"]
        loss = g.add(loss, g.policyLoss(X, t, g.array(old), g.array(adv), g.array(ref), None, (0.2, 0.2), 0.5))
    for k in range(300):
        g.zeroGrad()
        g.forward()
        g.backward(loss)
        if k % 100 == 99:
            np.testing.assert_allclose(X.grad, want, rtol=0, atol=2 * U * np.abs(want).max())
    # and added to what earlier passes left, as every gradient is
    g.zeroGrad()
    for k in range(3):
        g.backward(loss)
    np.testing.assert_allclose(X.grad, 3 * want, rtol=0, atol=8 * U * np.abs(want).max())


def test_a_refused_op_leaves_the_tape(ops, G):
    """Settings that the entry point refuses, and an arena that is full: the tape is what it was, runs again and gives the same gradients."""
    from znn_b200._lib import ZnnError
    x, t, old, adv, ref = case(12)
    want = ops.policy_loss(x, t, old, adv)["dlogits"]
    g = G(320 << 10)
    X, o, a = g.array(x, True), g.array(old), g.array(adv)
    loss = g.policyLoss(X, t, o, a)
    L = g.tokenLogProb(X, t)
    n = g.num_ops()
    for refused in (lambda: g.policyLoss(X, t, o, a, kl_coef=0.1), lambda: g.policyLoss(X, t, o, a, clip=(2.0, 0.2)), lambda: g.policyLoss(X, t, o, a, inv_temp=0.0),
                    lambda: g.tokenLogProb(X, t, -1.0), lambda: g.preferenceLoss(L, [0, 3, 9], beta=np.nan), lambda: g.preferenceLoss(L, [0, 3, 9], label_smoothing=1.0)):
        with pytest.raises(ZnnError):
            refused()
        assert g.num_ops() == n
    g.forward()
    g.backward(loss)
    np.testing.assert_array_equal(X.grad, want)
    with pytest.raises(ZnnError, match="arena"):
        for _ in range(10000):
            g.policyLoss(X, t, o, a)
            n += 1
    assert g.num_ops() == n
    with pytest.raises(ZnnError, match="arena"):
        for _ in range(10000):
            g.tokenLogProb(X, t)
            n += 1
    assert g.num_ops() == n
    g.forward()


def test_integers_of_graph_ops_and_models(ops, G):
    """Targets and row numbers travel as doubles: what is no 32-bit integer is refused, not cast to a row that is left out."""
    from znn_b200._lib import ZnnError
    from znn_b200.models import Model
    x, t, old, adv, _ = case(13, M=6)
    g = G()
    X, o, a = g.array(x, True), g.array(old), g.array(adv)
    L = g.tokenLogProb(X, t)
    for bad in (3e9, -3e9, 1.5, np.nan, np.inf):
        b = list(t[:-1]) + [bad]
        for f in (lambda: g.tokenLogProb(X, b), lambda: g.policyLoss(X, b, o, a), lambda: g.preferenceLoss(L, [0, 3, 6], None, b), lambda: g.preferenceLoss(L, [0, 3, bad])):
            with pytest.raises(ZnnError, match="32-bit integer"):
                f()
    m = Model("gpt", (67, 24, 32, 2, 1), arena_bytes=64 << 20)
    ids = np.zeros((2, 5), np.float32)
    wide = np.full((2, 5), 2 ** 32 + 3)
    for f in (lambda: m.token_logprobs(ids, wide), lambda: m.policy_step(ids, wide, ids, ids), lambda: m.preference_step(ids, wide)):
        with pytest.raises(ValueError, match="32-bit"):
            f()
    assert np.all(m.token_logprobs(ids, np.full((2, 5), 3)) < 0)
