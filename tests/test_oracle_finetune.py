"""The float64 checker of the fine-tuning operators against differences of its own losses."""
import numpy as np
import pytest

from oracle import finetune as ft


def differences(f, x, h=1e-6):
    g = np.zeros_like(x)
    for i in np.ndindex(x.shape):
        a, b = x.copy(), x.copy()
        a[i] += h
        b[i] -= h
        g[i] = (f(a) - f(b)) / (2 * h)
    return g


def inputs(seed, M=6, N=9):
    r = np.random.default_rng(seed)
    x = r.standard_normal((M, N)) * 1.5
    t = r.integers(0, N, M)
    t[2] = -1
    return r, x, t


# central differences of a smooth function of size ~1: truncation h^2 and rounding 1e-16 / h, both below 1e-9; 1e-8 leaves room
@pytest.mark.parametrize("inv_temp", [1.0, 0.6])
def test_log_probability_and_entropy(inv_temp):
    r, x, t = inputs(1)
    g, h = r.standard_normal(6), r.standard_normal(6)

    def f(v):
        logp, ent = ft.rows(v, t, inv_temp)[:2]
        return float((g * logp)[t >= 0].sum() + (h * ent)[t >= 0].sum())
    np.testing.assert_allclose(ft.rows_grad(x, t, g, h, inv_temp), differences(f, x), atol=1e-8)


@pytest.mark.parametrize("kl,ce,weighted", [(0.0, 0.0, False), (0.3, 0.0, False), (0.0, 0.2, True), (0.1, 0.05, True)])
def test_policy_loss(kl, ce, weighted):
    r, x, t = inputs(2, M=12)
    logp = ft.rows(x, t, 0.8)[0]
    old, ref, adv = logp - r.choice([-0.5, -0.1, 0.1, 0.5], 12), logp + 0.2 * r.standard_normal(12), r.standard_normal(12)
    w = r.random(12) if weighted else None
    f = lambda v: ft.policy(v, t, old, adv, ref, w, (0.2, 0.3), kl, ce, 0.8)["loss"]   # noqa: E731
    np.testing.assert_allclose(ft.policy(x, t, old, adv, ref, w, (0.2, 0.3), kl, ce, 0.8)["dlogits"], differences(f, x), atol=1e-8)


@pytest.mark.parametrize("by_length", [False, True])
def test_preference_loss(by_length):
    r = np.random.default_rng(3)
    off, t = [0, 4, 4, 9, 13], np.where(np.arange(15) % 5 == 3, -1, 1)
    logp, ref = -r.random(15) * 3, -r.random(15) * 3
    f = lambda v: ft.preference(v, off, ref, t, 0.7, 0.1, 0.2, by_length)["loss"]   # noqa: E731
    np.testing.assert_allclose(ft.preference(logp, off, ref, t, 0.7, 0.1, 0.2, by_length)["dlogp"], differences(f, logp), atol=1e-8)


def test_limits_of_infinite_losses():
    """A target whose log-probability is -inf: the KL term's limit is +inf, its slope -inf; a switched-off column has gradient 0."""
    x = np.array([[0.5, -np.inf, 1.0, -np.inf]])
    out = ft.policy(x, np.array([1]), [-1.0], [1.0], ref=[-2.0], kl=0.1)
    assert out["loss"] == np.inf and out["token_loss"][0] == np.inf
    np.testing.assert_array_equal(out["dlogits"], [[np.inf, -np.inf, np.inf, 0.0]])
    out = ft.policy(np.full((1, 4), -np.inf), np.array([1]), [-1.0], [1.0], ref=[-2.0], kl=0.1)
    assert out["loss"] == np.inf and np.all(out["dlogits"] == 0.0)


def test_limits_of_infinite_margins():
    inf = np.inf
    for smooth, losses in ((0.0, [0.0, inf]), (0.1, [inf, inf])):
        out = ft.preference([-1.0, -inf, -inf, -1.0], [0, 1, 2, 3, 4], beta=0.5, smoothing=smooth)
        np.testing.assert_array_equal(out["pair_loss"], losses)
        np.testing.assert_allclose(out["dlogp"], np.array([smooth, -smooth, smooth - 1, 1 - smooth]) * 0.25, atol=1e-15)
