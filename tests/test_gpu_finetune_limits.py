"""The fine-tuning operators where values leave the ordinary range: terms that cancel, infinite log-probabilities, rows that are
nearly certain, norms beyond any bound.  Against float64 forms that keep what those rows are about; U = 2^-24 is half a step of fp32,
K (row_k) the error of a row's sum in such halves, as test_gpu_finetune.py derives them."""
import ctypes as C

import numpy as np
import pytest

import test_gpu_finetune as base
from oracle import finetune as ft
from test_gpu_finetune import INF, U, row_k, within

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    from znn_b200 import ops as _ops
    _ops.init(0)
    return _ops


@pytest.fixture(scope="module")
def L(ops):
    from znn_b200._lib import lib
    return lib()


# ------------------------------------------------------------------ the KL term where its parts cancel
@pytest.mark.parametrize("N", [1, 8, 64, 512, 2048, 16384])
def test_kl_term_alone(ops, N):
    """Rows of N = 2^k equal logits have logp = -k log 2, which the operator has in fp64, so q = ref - logp is known to its own
    rounding, and with an advantage of 0 the row's loss is kl_coef * (e^q - q - 1) alone.  Errors in halves of a step: q is rounded
    to fp32, which moves the term by |q (e^q - 1)|; the series below 1/2 in size has a square, a product and sums whose last
    rounds 0.5 + ..., together 4 of the term; above, expm1f is off by 2 of its value (its documented step) and the difference by 1 of
    the term; kl_coef's product and nothing else comes after that: 1."""
    q = np.exp(np.linspace(np.log(1e-4), np.log(8.0), 500))
    q = np.concatenate([q, -q])
    logp = -np.log(np.float64(N))
    ref = (logp + q).astype(np.float32)
    q = ref.astype(np.float64) - logp
    M, kl = len(q), float(np.float32(0.1))
    x = np.full((M, N), 0.25, np.float32)
    got = ops.policy_loss(x, np.zeros(M, np.int32), np.full(M, logp, np.float32), np.zeros(M, np.float32), ref, None, (0.2, 0.2), kl)
    e = np.expm1(q)
    small = np.abs(q) < 0.6
    # e^q - q - 1 in float64 from its series where q is small: expm1(q) - q would leave 1e-12 of it
    series = sum(q ** k / np.prod(np.arange(1.0, k + 1)) for k in range(2, 25))
    want = kl * np.where(small, series, e - q)
    within(got["token_loss"], want, U * (kl * (np.abs(q * e) + np.where(np.abs(q) < 0.5, 0.0, 2 * np.abs(e))) + 5 * want), "kl_coef * (e^q - q - 1)")


# ------------------------------------------------------------------ infinite losses
@pytest.mark.parametrize("N", [6, 40, 300, 900, 1500, 5001, 20000, 131072])
@pytest.mark.parametrize("kl,ce", [(0.1, 0.0), (0.1, 0.05), (0.0, 0.0), (0.0, 0.05)])
def test_infinite_policy_losses(ops, N, kl, ce):
    """A target that is switched off, a row with no logit at all, and differences whose exponential is beyond fp32: the loss is +inf (KL
    term, or a loss of an unbounded ratio), columns that are switched off have gradient 0, the others of the row +-inf; a row with no
    logit has gradient 0; the rows beside them are as ever."""
    r = np.random.default_rng(N)
    M = 7
    x = r.standard_normal((M, N)).astype(np.float32)
    off = np.zeros((M, N), bool)
    off[:, 2] = True
    if N > 40:
        off[:, N // 2:N // 2 + N // 8] = True
    x[off] = -INF
    t = np.array([0, 2, 1, N - 1, 1, 0, 2], np.int32)
    x[2] = -INF
    clean = np.zeros((M, N), np.float32)
    clean[:] = x
    clean[[1, 2, 6]] = 0.0
    logp = ft.rows(clean, np.where(np.isin(np.arange(M), [1, 2, 6]), 0, t))[0]
    old, ref = (logp - 0.1).astype(np.float32), (logp + 0.2).astype(np.float32)
    adv = np.array([0.7, 1.0, -1.0, 0.5, -2.0, 0.3, 0.0], np.float32)
    ref[3] = 95.0                      # q above 88.7
    old[4] = -150.0                    # the ratio, with an advantage that does not bound it
    out = ops.policy_loss(x, t, old, adv, ref if kl else None, None, (0.2, 0.2), float(np.float32(kl)), float(np.float32(ce)))
    infinite = np.array([False, kl > 0, kl > 0, kl > 0, True, False, kl > 0])
    assert np.all(out["token_loss"][infinite] == INF), out["token_loss"]
    assert np.all(np.isfinite(out["token_loss"][~infinite])), out["token_loss"]
    assert out["loss"] == INF and out["rows"] == M
    dx = out["dlogits"]
    hot = np.arange(N)[None] == t[:, None]
    assert np.all(dx[2] == 0.0)
    assert np.all(dx[off & ~hot] == 0.0)
    for i in np.flatnonzero(infinite):
        if i == 2:
            continue
        # KL: the gradient asks for a larger log-probability; an unbounded ratio with a negative advantage for a smaller one
        sign = 1.0 if i == 4 else -1.0
        assert np.all(dx[i][~off[i] & ~hot[i]] == -sign * INF), dx[i]
        assert dx[i, t[i]] == sign * INF, dx[i, t[i]]
    fine = np.flatnonzero(~infinite)
    alone = ops.policy_loss(x[fine], t[fine], old[fine], adv[fine], ref[fine] if kl else None, np.full(len(fine), 1 / M, np.float32), (0.2, 0.2),
                            float(np.float32(kl)), float(np.float32(ce)))
    # (the weight 1 / M is made by the same fp32 division)
    np.testing.assert_array_equal(dx[fine], alone["dlogits"])
    np.testing.assert_array_equal(out["token_loss"][fine], alone["token_loss"])


def test_a_certain_token_with_an_infinite_ratio_has_no_gradient(ops):
    """p = 1 at the target and nothing beside it: 1 - p and every other p_j are 0, whatever the slope"""
    for N in (5, 200, 700, 3000, 40000):
        x = np.full((1, N), -INF, np.float32)
        x[0, N - 2] = 3.0
        out = ops.policy_loss(x, np.array([N - 2], np.int32), np.array([-120.0], np.float32), np.array([-1.0], np.float32))
        assert out["token_loss"][0] == INF and out["logp"][0] == 0.0 and np.all(out["dlogits"] == 0.0)


@pytest.mark.filterwarnings("ignore:invalid value")   # inf - inf in the comparison of equal infinities
@pytest.mark.parametrize("P,length", [(4, 5), (40, 30), (4, 3000), (2, 20000)])
@pytest.mark.parametrize("smooth", [0.0, 0.1])
@pytest.mark.parametrize("by_length", [False, True])
def test_infinite_rewards(ops, P, length, smooth, by_length):
    """A log-probability of -inf in the other answer (margin +inf: loss 0, or +inf where labels are smoothed), in the preferred one
    (margin -inf: loss +inf, slope 1 - label_smoothing), in both (no margin: NaN); an ordinary pair beside them."""
    r = np.random.default_rng(P)
    M = 2 * P * length
    logp = (-2 * r.random(M)).astype(np.float32)
    off = (np.arange(2 * P + 1) * length).astype(np.int32)
    logp[1 * length + 2] = -INF                      # pair 0: the other answer
    logp[2 * length + 1] = -INF                      # pair 1: the preferred one
    beta, smooth = float(np.float32(0.3)), float(np.float32(smooth))
    got = ops.preference_loss(logp, off, None, None, beta, smooth, 0.0, by_length)
    want = ft.preference(logp, off, None, None, beta, smooth, 0.0, by_length)
    share = beta / length if by_length else beta
    assert want["pair_loss"][0] == (np.inf if smooth else 0.0) and want["pair_loss"][1] == np.inf
    np.testing.assert_allclose(want["dlogp"][:length], smooth / P * share, rtol=1e-12)
    np.testing.assert_allclose(want["dlogp"][2 * length:3 * length], (smooth - 1) / P * share, rtol=1e-12)
    # as test_preference_loss: fp64 inside, one rounding of each output
    for k in ("pair_loss", "rewards", "dlogp"):
        within(got[k], want[k], U * np.abs(np.where(np.isfinite(want[k]), want[k], 0.0)) * 1.001 + 1e-12, k)
    assert got["loss"] == INF
    if P > 2:
        logp[2 * length + 1] = -1.0
        got = ops.preference_loss(logp, off, None, None, beta, 0.0, 0.0, by_length)
        want = ft.preference(logp, off, None, None, beta, 0.0, 0.0, by_length)
        assert np.isfinite(want["loss"])
        within(got["loss"], want["loss"], 2 * U * want["loss"] * 1.001 + 1e-12, "loss")
        logp[4 * length] = logp[5 * length] = -INF
        got = ops.preference_loss(logp, off, None, None, beta, 0.0, 0.0, by_length)
        assert np.isnan(got["loss"]) and np.isnan(got["pair_loss"][2]) and np.all(np.isfinite(np.delete(got["pair_loss"], 2)))


# ------------------------------------------------------------------ rows that are nearly certain
def nearly_certain(r, sigma, N, top, shift):
    """A row whose largest logit stands at `top` and whose others' exponentials sum to about sigma, relative to the largest"""
    d = np.minimum(np.log(sigma / max(N - 1, 1)) + 0.5 * r.standard_normal(N), -0.2)
    x = (shift + d).astype(np.float32)
    x[top] = shift
    return x


def certain_case(N, seed, inv_temp):
    """sums of the others from 0.7 down to 1e-9, the target at the largest logit or (every fourth row) elsewhere; float64 scalars that
    keep the small part"""
    r = np.random.default_rng(seed)
    sigma = np.repeat([0.7, 0.3, 0.2, 0.05, 1e-2, 1e-3, 1e-4, 1e-6, 1e-9], 4)
    M = len(sigma)
    top = r.integers(0, N, M)
    x = np.stack([nearly_certain(r, s ** (1 / inv_temp), N, k, np.float32(r.uniform(-8, 8))) for s, k in zip(sigma, top)])
    t = np.where(np.arange(M) % 4 == 3, (top + 1 + r.integers(0, N - 1, M)) % N, top).astype(np.int32)
    d = (x.astype(np.float64) - x[np.arange(M), top].astype(np.float64)[:, None]) * inv_temp
    e = np.exp(d)
    e[np.arange(M), top] = 0.0                       # the others alone
    small = e.sum(1)
    log_s = np.log1p(small)
    p = e / (1 + small)[:, None]
    u = (p * d).sum(1)
    return r, x, t, top, d, small, log_s, p, u, log_s - u


SIZES = [2, 5, 33, 64, 65, 300, 400, 512, 700, 1000, 1025, 5000, 8191, 8192, 9001, 40000]


@pytest.mark.parametrize("N", SIZES)
@pytest.mark.parametrize("inv_temp", [1.0, 0.8])
def test_log_probabilities_of_nearly_certain_rows(ops, N, inv_temp):
    """logp and entropy to a few K halves of a step of their own value, however small: every exponential carries 2 D + 4, the sums
    N / 32 + 16 (K), log1p and the division 2 more each; -u (positive) is made of products d e with 3 more; nothing cancels at the
    largest logit.  Elsewhere logp is d - log s, of size |logp|."""
    inv_temp = float(np.float32(inv_temp))
    r, x, t, top, d, small, log_s, p, u, H = certain_case(N, N, inv_temp)
    K = row_k(x, inv_temp) + 8
    logp, ent, _ = ops.token_logprob_fwd(x, t, inv_temp)
    want = np.where(t == top, -log_s, d[np.arange(len(t)), t] - log_s)
    tol = np.where(t == top, K, 4) * U * np.abs(want) + np.where(t == top, 0.0, K * U * log_s)
    within(logp, want, tol, "logp")
    within(ent, H, K * U * H, "entropy")
    out = ops.policy_loss(x, t, want.astype(np.float32), np.ones(len(t), np.float32), inv_temp=inv_temp)
    within(out["logp"], want, tol, "logp of the policy loss")


@pytest.mark.parametrize("N", SIZES)
@pytest.mark.parametrize("entropy", [False, True])
@pytest.mark.parametrize("accumulate,in_place", [(False, False), (True, False), (False, True)])
def test_gradient_of_nearly_certain_rows(ops, L, N, entropy, accumulate, in_place):
    """inv_temp (g ([j = t] - p_j) - h p_j (log p_j + H)), each part to K + 24 halves of a step of its own size.  At the largest logit
    1 - p is the others' sum over the whole, and log p + H = -u; where the others sum to 1/32 or more, 1 - p is a difference of
    fp32 numbers, which leaves 3 halves of a step of p (the sum's, the quotient's, the exponential's)."""
    inv_temp = float(np.float32(0.8))
    r, x, t, top, d, small, log_s, p, u, H = certain_case(N, N + 1, inv_temp)
    M, rows = len(t), np.arange(len(t))
    _, ent, stats = ops.token_logprob_fwd(x, t, inv_temp)
    g, h = r.standard_normal(M).astype(np.float32), (r.standard_normal(M) * entropy).astype(np.float32)
    part = p.copy()
    part[rows, top] = 1 / (1 + small)
    hot = np.zeros((M, N))
    hot[rows, t] = 1.0
    one_less = hot - part
    one_less[rows, top] = np.where(t == top, small / (1 + small), -1 / (1 + small))
    inner = part * (d - log_s[:, None] + H[:, None])
    size = part * (np.abs(d) + log_s[:, None] + H[:, None])
    inner[rows, top] = part[rows, top] * -u
    size[rows, top] = part[rows, top] * (H + log_s)
    G, E = g.astype(np.float64)[:, None], h.astype(np.float64)[:, None]
    want = inv_temp * (G * one_less - E * inner)
    tol = inv_temp * (np.abs(G) * np.abs(one_less) + np.abs(E) * size) * (row_k(x, inv_temp)[:, None] + 24) * U
    tol += inv_temp * 3 * U * np.abs(G) * (part * hot) * (small >= 1 / 32.01)[:, None]
    before = (r.standard_normal((M, N)) * small[:, None]).astype(np.float32)
    if in_place:
        up = ops.DevBuf.from_host
        xb, tb, sb, gb, eb, hb = up(x), up(t), up(stats), up(g), up(ent), up(h)
        L.call("znn_token_logprob_bwd", xb.ptr, N, tb.ptr, inv_temp, sb.ptr, eb.ptr if entropy else None, gb.ptr, hb.ptr if entropy else None, xb.ptr, N, 0, M, N)
        got = xb.to_host((M, N))
        apart = ops.token_logprob_bwd(x, t, stats, g, None, ent if entropy else None, h if entropy else None, inv_temp)
        np.testing.assert_array_equal(got, apart)
    else:
        got = ops.token_logprob_bwd(x, t, stats, g, before.copy() if accumulate else None, ent if entropy else None, h if entropy else None, inv_temp)
    if accumulate:
        want = want + before
    within(got, want, tol + U * np.abs(want), "dlogits")


# ------------------------------------------------------------------ norms beyond any bound
@pytest.mark.parametrize("n", [5, 5000, 2000003])
def test_a_factor_below_fp32_is_not_a_skipped_step(ops, n):
    """A finite norm so far above the bound that their quotient is below fp32: the gradients are clipped (by the smallest factor there
    is), not left as they are as if the norm were not finite."""
    value = np.float32(3e38)
    for big in (1, n):                                   # a norm within fp32, and one beyond it
        g = np.zeros(n, np.float32)
        g[:big] = value
        norm = float(value) * np.sqrt(big)
        got = ops.clip_grads([g], 1e-20)
        assert got[0] == np.float32(norm) if norm < 3.4e38 else got[0] == INF
        assert 0 < got[1] <= 2.0 ** -149
        np.testing.assert_array_equal(g[:big], value * got[1])
        w = np.full(n, 0.5, np.float32)
        ops.sgd_step_clipped(w, np.where(np.arange(n) < big, value, 0).astype(np.float32), None, 1.0, 0.0, 1e-20)
        assert np.all(w[:big] < 0.5) and np.all(np.isfinite(w))


# ------------------------------------------------------------------ the policy loss that makes no entropies
class WithoutEntropies:
    """ops, with policy losses as a step without an entropy term calls them: no buffer for entropies.  Those that the caller compares
    come from a call of their own."""

    def __init__(self, ops):
        self.ops = ops

    def policy_loss(self, *args, **kw):
        out = self.ops.policy_loss(*args, want_entropy=False, **kw)
        assert out["entropy"] is None
        kw["want_grad"] = False
        out["entropy"] = self.ops.policy_loss(*args, **kw)["entropy"]
        return out


MANY = [(450, 1100), (520, 1501), (450, 2000), (451, 2100), (450, 2900), (450, 5121), (447, 6000), (450, 9001), (450, 12500), (300, 51300), (160, 110000)]


@pytest.mark.parametrize("M,N", base.SHAPES + MANY)
@pytest.mark.parametrize("kl,weighted,inv_temp", [(0.0, False, 1.0), (0.05, False, 1.25), (0.1, True, 0.7)])
def test_policy_loss_without_entropies(ops, M, N, kl, weighted, inv_temp):
    base.test_policy_loss(WithoutEntropies(ops), M, N, kl, 0.0, weighted, inv_temp)


# ------------------------------------------------------------------ rows of every kind in one call
@pytest.mark.parametrize("N", [1, 7, 31, 33, 64, 65, 100, 128, 129, 200, 257, 384, 385, 513, 700, 1025, 5000, 9001])
@pytest.mark.parametrize("accumulate,in_place", [(False, False), (True, False), (False, True)])
@pytest.mark.parametrize("shift", [0, 1])
def test_gradients_of_rows_among_others_and_alone(ops, L, N, accumulate, in_place, shift):
    """Nearly certain rows, others, rows that are left out, empty ones and bad targets share warps: each gives the bits that it gives
    alone, and the floats between the rows and behind the last one stay."""
    r = np.random.default_rng(N * 2 + shift)
    M, ld = 75, N + (3 if shift else 4)
    x = (r.standard_normal((M, N)) * 2).astype(np.float32)
    t = r.integers(0, N, M).astype(np.int32)
    certain = r.random(M) < 0.4
    x[certain, r.integers(0, N, M)[certain]] += 30.0
    target_at_top = r.random(M) < 0.7
    t[target_at_top] = x.argmax(1)[target_at_top]
    x[r.random(M) < 0.05] = -INF
    t[r.random(M) < 0.15] = -1
    t[r.random(M) < 0.05] = N + 3
    g, h = r.standard_normal(M).astype(np.float32), r.standard_normal(M).astype(np.float32)
    logp, ent, stats = ops.token_logprob_fwd(x, t)
    base.status(L)
    up = ops.DevBuf.from_host

    def spread(a):
        buf = np.full(shift + M * ld + 16, 77.0, np.float32)
        for i in range(M):
            buf[shift + i * ld:shift + i * ld + N] = a[i]
        return buf
    hx, before = spread(x), spread(r.standard_normal((M, N)).astype(np.float32))
    tb, sb, gb, hb, eb = up(t), up(stats), up(g), up(h), up(ent)

    def run(xb, db, first, rows, entropy):
        L.call("znn_token_logprob_bwd", xb.ptr + 4 * (shift + first * ld), ld, tb.ptr + 4 * first, 1.0, sb.ptr + 8 * first, eb.ptr + 4 * first if entropy else None,
               gb.ptr + 4 * first, hb.ptr + 4 * first if entropy else None, db.ptr + 4 * (shift + first * ld), ld, int(accumulate), rows, N)
    for entropy in (False, True):
        x1, x2, d1, d2 = up(hx), up(hx), up(before), up(before)
        a, b = (x1, x2) if in_place else (d1, d2)
        run(x1, a, 0, M, entropy)
        for i in range(M):
            run(x2, b, i, 1, entropy)
        together, alone = a.to_host(hx.shape), b.to_host(hx.shape)
        np.testing.assert_array_equal(together, alone)
        rest = together.copy()
        for i in range(M):
            row = rest[shift + i * ld:shift + i * ld + N]
            assert np.all(np.isfinite(row))
            if not 0 <= t[i] < N or stats[i, 1] == 0:
                np.testing.assert_array_equal(row, before[shift + i * ld:shift + i * ld + N] if accumulate else 0.0)
            row[:] = 77.0
        assert np.all(rest == 77.0)
        if not in_place:
            np.testing.assert_array_equal(x1.to_host(hx.shape), hx)
