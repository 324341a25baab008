"""Token log-probabilities, policy loss, preference loss and gradient clipping on the GPU against float64 (oracle/finetune.py).

Tolerances count roundings of u = 2^-24 (half a step of fp32), derived as follows.  A distance d = inv_temp * (x - xm) carries
two roundings, 2u|d| <= 2u D with D the largest |d| whose exponential is not 0 (at most 104); exp() is good to 2 of its own
steps = 4u; a sum of N positive terms over at least 32 lanes with at most N / 32 additions in a row, and 16 in the joins, is
good to (N / 32 + 16) u.  So log s is good to K u with K = 2 D + 4 + N / 32 + 16, and everything that is made of p or log p to
a small multiple of it, which each function below writes out.  What comes out in fp32 is rounded once more: u of its value."""
import ctypes as C

import numpy as np
import pytest

from oracle import finetune as ft

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
INF = np.float32(np.inf)


@pytest.fixture(scope="module")
def ops():
    from znn_b200 import ops as _ops
    _ops.init(0)
    return _ops


@pytest.fixture(scope="module")
def L(ops):
    from znn_b200._lib import lib
    return lib()


def status(L):
    st = C.c_int(0)
    L.call("znn_device_status", C.byref(st), 1)
    return st.value


def within(got, want, tol, what):
    got, want = np.asarray(got, np.float64), np.asarray(want, np.float64)
    tol = np.broadcast_to(np.asarray(tol, np.float64), want.shape)
    assert got.shape == want.shape, what
    special = ~np.isfinite(want)
    same = np.where(np.isnan(want), np.isnan(got), got == want)
    assert np.all(same[special]), f"{what}: {got[special][:4]} instead of {want[special][:4]}"
    err = np.abs(got - want)[~special]
    ok = err <= tol[~special]
    assert np.all(ok), f"{what}: off by {err[~ok][:4]}, allowed {tol[~special][~ok][:4]}, at {want[~special][~ok][:4]} ({(~ok).sum()} of {ok.size})"


def row_k(x, inv_temp):
    """K of the head of this file, per row"""
    x = np.asarray(x, np.float64)
    fin = np.where(np.isfinite(x), x, np.nan)
    with np.errstate(all="ignore"):
        spread = np.nanmax(fin, 1, initial=-1e300) - np.nanmin(fin, 1, initial=1e300)
    D = np.minimum(np.where(np.isfinite(spread) & (spread > 0), spread, 0.0) * inv_temp, 104.0)
    return 2 * D + 20 + x.shape[1] / 32


def logits(r, M, N, banned=True, left=0.2):
    x = (r.standard_normal((M, N)) * 2.5).astype(np.float32)
    if banned and N > 4:
        x[r.random((M, N)) < 0.1] = -INF
    t = r.integers(0, N, M).astype(np.int32)
    x[np.arange(M), t] = (r.standard_normal(M) * 2 + 4).astype(np.float32)
    out = r.random(M) < left
    x[out] = np.nan        # what a row that is left out holds must not matter
    t[out] = -1
    return x, t


SHAPES = [(1, 1), (3, 2), (5, 10), (33, 31), (17, 32), (40, 255), (9, 1000), (7, 1021), (4, 1024), (6, 1025), (5, 2047), (3, 4096),
          (5, 4099), (3, 8191), (20, 8192), (3, 8193), (2, 16384), (3, 16389), (2, 32003), (2, 50257), (1, 131072), (1, 140001), (1, 300007),
          (300, 7), (1000, 130), (150, 8192)]


@pytest.mark.parametrize("M,N", SHAPES)
@pytest.mark.parametrize("inv_temp", [1.0, 0.7])
def test_token_logprob(ops, M, N, inv_temp):
    r = np.random.default_rng(M * 1000 + N)
    inv_temp = float(np.float32(inv_temp))
    x, t = logits(r, M, N)
    logp, ent, stats = ops.token_logprob_fwd(x, t, inv_temp)
    used = t >= 0
    xs = np.where(used[:, None], x, 0.0)
    lw, ew, p, lp, _, _ = ft.rows(xs, t, inv_temp)
    K = row_k(xs, inv_temp)
    within(logp, lw, K * U + U * np.abs(lw), "logp")
    # H = log s - u / s: u / s = -E|d| carries the error of each d, of exp, of the sums and of the quotient
    spread = np.where(p > 0, p * np.abs(np.where(np.isfinite(lp), lp, 0.0)), 0.0).sum(1) + np.abs(np.log(np.maximum(stats[:, 1], 1)))
    within(ent, ew, (K * (1 + 2 * spread) + 4) * U + U * ew, "entropy")
    top = np.where(used, xs.max(1), 0.0)
    within(stats[:, 0], top, 0.0, "row maximum")
    with np.errstate(invalid="ignore"):
        s = np.where(used, np.exp((xs.astype(np.float64) - xs.max(1, keepdims=True)) * inv_temp).sum(1), 0.0)
    within(stats[:, 1], s, (K + 1) * U * s, "row sum")
    none = ops.token_logprob_fwd(x, t, inv_temp, want_entropy=False)
    np.testing.assert_array_equal(none[0], logp)
    np.testing.assert_array_equal(none[2], stats)


def grad_tolerance(x, t, p, lp, ent, g, h, inv_temp, more):
    """p carries K u, log p + H another K u (1 + |log p| + H); the coefficients `more` (relative); 8 roundings on the way."""
    K = row_k(x, inv_temp)[:, None] + 8 + more
    hot = np.zeros_like(p)
    hot[np.arange(len(t)), np.maximum(t, 0)] = 1.0
    inner = p * (2 + 2 * np.abs(np.where(p > 0, lp, 0.0)) + 2 * np.abs(ent[:, None]))
    return U * inv_temp * K * (np.abs(g)[:, None] * (hot + p) + np.abs(h)[:, None] * (inner + hot * 0))


@pytest.mark.parametrize("M,N", SHAPES)
@pytest.mark.parametrize("entropy,accumulate", [(False, False), (True, False), (True, True), (False, True)])
def test_token_logprob_grad(ops, M, N, entropy, accumulate):
    r = np.random.default_rng(M * 1000 + N + 1)
    inv_temp = float(np.float32(0.8))
    x, t = logits(r, M, N)
    used = t >= 0
    xs = np.where(used[:, None], x, 0.0)
    _, ent, p, lp, _, _ = ft.rows(xs, t, inv_temp)
    top = np.where(used, xs.max(1), 0.0)
    with np.errstate(invalid="ignore"):
        s = np.where(used, np.exp((xs.astype(np.float64) - xs.max(1, keepdims=True)) * inv_temp).sum(1), 0.0)
    stats = np.stack([top, s], 1).astype(np.float32)
    g, h = r.standard_normal(M).astype(np.float32), r.standard_normal(M).astype(np.float32)
    g[~used] = np.nan
    h[~used] = np.nan
    before = r.standard_normal((M, N)).astype(np.float32) if accumulate else None
    got = ops.token_logprob_bwd(x, t, stats, g, before.copy() if accumulate else None, ent.astype(np.float32) if entropy else None,
                                h if entropy else None, inv_temp)
    gz, hz = np.where(used, g, 0.0).astype(np.float64), np.where(used, h if entropy else 0.0, 0.0).astype(np.float64)
    want = ft.rows_grad(xs, t, gz, hz, inv_temp)
    tol = grad_tolerance(xs, t, p, lp, ent, gz, hz, inv_temp, 0)
    if accumulate:
        np.testing.assert_array_equal(got[~used], before[~used])
        want = want + before
    within(got, want, tol + U * np.abs(want), "dlogits")
    if not accumulate:
        assert np.all(got[~used] == 0.0)


def policy_case(r, M, N, inv_temp, clip):
    x, t = logits(r, M, N)
    if M > 2:
        t[0], x[0] = 0, r.standard_normal(N).astype(np.float32)
    used = t >= 0
    xs = np.where(used[:, None], x, 0.0)
    logp = ft.rows(xs, t, inv_temp)[0]
    # ratios on both sides of both borders, none within 1e-3 of one: there the gradient jumps
    ratio = r.choice([0.5, 1 - clip[0] - 0.01, 1 - clip[0] + 0.01, 1.0, 1 + clip[1] - 0.01, 1 + clip[1] + 0.01, 1.9], M)
    old = (logp - np.log(ratio)).astype(np.float32)
    ref = (logp + 0.4 * r.standard_normal(M)).astype(np.float32)
    adv = r.standard_normal(M).astype(np.float32)
    adv[r.random(M) < 0.1] = 0.0
    for a in (old, ref, adv):
        a[~used] = np.nan
    return x, xs, t, used, old, ref, adv


def check_policy(got, want, xs, t, used, old, ref, adv, clip, kl, ce, inv_temp, grad=True):
    logp, ent, p, lp, _, _ = ft.rows(xs, t, inv_temp)
    K = row_k(xs, inv_temp)
    off_logp = K * U                       # of the fp64 log-probability that ratio and q are made of
    spread = np.where(p > 0, p * np.abs(np.where(np.isfinite(lp), lp, 0.0)), 0.0).sum(1) + np.abs(np.where(used, logp, 0.0)) + 20
    off_ent = (K * (1 + 2 * spread) + 4) * U
    o, f, a = (np.where(used, v, 0.0).astype(np.float64) for v in (old, ref, adv))
    with np.errstate(over="ignore", invalid="ignore"):
        ratio, q = np.exp(logp - o), f - logp
        slope = np.abs(a) * ratio + kl * (np.exp(q) + 1)
    tok = want["token_loss"]
    within(got["logp"], want["logp"], off_logp + U * np.abs(want["logp"]), "logp")
    within(got["entropy"], want["entropy"], off_ent + U * want["entropy"], "entropy")
    tol_tok = off_logp * slope + ce * off_ent + U * np.abs(np.where(np.isfinite(tok), tok, 0.0))
    within(got["token_loss"], tok, tol_tok, "token_loss")
    assert got["rows"] == want["rows"]
    return off_logp, off_ent, slope, tol_tok, (p, lp, ent, logp)


@pytest.mark.parametrize("M,N", SHAPES)
@pytest.mark.parametrize("kl,ce,weighted,inv_temp", [(0.0, 0.0, False, 1.0), (0.05, 0.0, False, 1.25), (0.1, 0.02, True, 0.7), (0.0, 0.3, True, 1.0)])
def test_policy_loss(ops, M, N, kl, ce, weighted, inv_temp):
    r = np.random.default_rng(M * 1000 + N + 2)
    kl, ce, inv_temp, clip = float(np.float32(kl)), float(np.float32(ce)), float(np.float32(inv_temp)), (0.25, 0.5)
    x, xs, t, used, old, ref, adv = policy_case(r, M, N, inv_temp, clip)
    w = None
    if weighted:
        w = (r.random(M) * 0.3 + 0.1).astype(np.float32)
        w[r.random(M) < 0.2] = 0.0
        adv[w == 0] = np.nan          # a row of weight 0 is left out like one without a target
    z = lambda v: np.where(used & (True if w is None else w != 0), v, 0.0)   # noqa: E731
    want = ft.policy(xs, t, z(old), z(adv), z(ref), w, clip, kl, ce, inv_temp)
    got = ops.policy_loss(x, t, old, adv, ref if kl else None, w, clip, kl, ce, inv_temp)
    use = used if w is None else used & (w != 0)
    off_logp, off_ent, slope, tol_tok, (p, lp, ent, logp) = check_policy(got, want, xs, np.where(use, t, -1), use, z(old), z(ref), z(adv), clip, kl, ce,
                                                                        inv_temp)
    ww = np.where(use, 1.0 / max(want["rows"], 1) if w is None else w, 0.0)
    within(got["loss"], want["loss"], float((ww * tol_tok).sum()) + 3 * U * float((ww * np.abs(want["token_loss"])).sum()) + U * abs(want["loss"]), "loss")
    # G = w * slope carries the error of logp twice (the ratio, or exp(q)); E = w * ce the rounding of w
    g, h = ww * np.where(use, slope, 0.0), ww * ce
    tol = grad_tolerance(xs, np.where(use, t, -1), p, lp, ent, g, h, inv_temp, 0) + inv_temp * (off_logp * np.where(use, slope, 0.0) * ww)[:, None] * 2 * (
        p + (np.arange(N)[None] == t[:, None])) + (off_ent * h)[:, None] * inv_temp * 2 * p
    # at the target the two parts are added in fp64 and rounded once
    hot = np.arange(N)[None] == t[:, None]
    tol = tol + hot * U * inv_temp * (h * (2 + np.abs(np.where(use, logp, 0.0)) + ent))[:, None] * row_k(xs, inv_temp)[:, None]
    within(got["dlogits"], want["dlogits"], tol + U * np.abs(want["dlogits"]), "dlogits")
    alone = ops.policy_loss(x, t, old, adv, ref if kl else None, w, clip, kl, ce, inv_temp, want_grad=False)
    for k in ("loss", "rows", "token_loss", "logp", "entropy"):
        np.testing.assert_array_equal(alone[k], got[k])


def test_policy_gradient_is_the_losses_slope(ops):
    """Against differences of the operator's own loss (fp32 inputs, fp64 sums): the step h = 2^-7 is exact in the logits; the
    central difference errs by h^2 / 6 times a third derivative below 4 (weights 1/5, |A| r below 3) = 5e-5, and by the loss's
    own error 1e-6 / h = 1.3e-4."""
    r = np.random.default_rng(5)
    M, N, h = 5, 6, 2.0 ** -7
    x = np.round(r.standard_normal((M, N)) * 64) .astype(np.float32) / 64
    t = r.integers(0, N, M).astype(np.int32)
    logp = ft.rows(x, t)[0]
    old, ref, adv = (logp - np.log([0.9, 1.6, 1.05, 0.5, 1.1])).astype(np.float32), (logp + 0.1).astype(np.float32), r.standard_normal(M).astype(np.float32)
    f = lambda v: float(ops.policy_loss(v, t, old, adv, ref, None, (0.2, 0.2), 0.1, 0.05, want_grad=False)["loss"])   # noqa: E731
    got = ops.policy_loss(x, t, old, adv, ref, None, (0.2, 0.2), 0.1, 0.05)["dlogits"]
    for i in np.ndindex(M, N):
        a, b = x.copy(), x.copy()
        a[i] += h
        b[i] -= h
        assert abs((f(a) - f(b)) / (2 * h) - got[i]) < 2e-4


# ------------------------------------------------------------------ rows and values at the edge
def test_rows_with_nothing_to_choose_from(ops):
    """-inf everywhere; -inf at the target; the type's lowest value as a mask"""
    N = 1030
    x = np.zeros((5, N), np.float32)
    x[0] = -INF
    x[1, :] = -INF
    x[1, 7] = 2.0                                  # one token left, and it is the target
    x[2, 3] = -INF                                 # the target is switched off
    x[3] = np.finfo(np.float32).min                # every logit masked by the lowest value: uniform
    x[4, 1:] = np.finfo(np.float32).min            # all but one masked by the lowest value
    t = np.array([5, 7, 3, 2, 0], np.int32)
    logp, ent, stats = ops.token_logprob_fwd(x, t)
    np.testing.assert_array_equal(stats[0], [-INF, 0.0])
    np.testing.assert_array_equal(logp[[0, 1, 2, 4]], np.array([-INF, 0.0, -INF, 0.0], np.float32))
    np.testing.assert_array_equal(ent[[0, 1, 4]], 0.0)
    within([logp[3], ent[3]], [-np.log(N), np.log(N)], 60 * U * np.log(N), "uniform")
    g = np.ones(5, np.float32)
    dx = ops.token_logprob_bwd(x, t, stats, g, entropy=ent, dentropy=g)
    assert np.all(np.isfinite(dx)) and np.all(dx[0] == 0.0) and np.all(dx[1] == 0.0) and dx[2, 3] == 1.0 and np.all(dx[4] == 0.0)
    # the policy loss on the same rows: ratio 0 where the token is impossible, no KL
    out = ops.policy_loss(x, t, np.full(5, -1, np.float32), np.ones(5, np.float32), entropy_coef=0.1)
    assert np.isfinite(out["loss"]) and np.all(np.isfinite(out["dlogits"])) and np.all(out["dlogits"][0] == 0.0)
    assert out["token_loss"][0] == 0.0


@pytest.mark.parametrize("N", [5, 300, 5000, 20000])
@pytest.mark.parametrize("value", [np.nan, np.inf])
def test_a_poisoned_row_stays_alone(ops, N, value):
    r = np.random.default_rng(N)
    x = r.standard_normal((3, N)).astype(np.float32)
    clean = x.copy()
    x[1, N - 2] = value
    t = np.array([0, 1, N - 1], np.int32)
    logp, ent, stats = ops.token_logprob_fwd(x, t)
    want = ops.token_logprob_fwd(clean, t)
    assert np.isnan(logp[1]) and np.isnan(ent[1])
    np.testing.assert_array_equal(logp[[0, 2]], want[0][[0, 2]])
    out = ops.policy_loss(x, t, want[0], np.ones(3, np.float32), entropy_coef=0.1)
    assert np.isnan(out["loss"]) and np.all(np.isfinite(out["dlogits"][[0, 2]])) and np.all(np.isnan(out["dlogits"][1]))


def test_targets_outside_the_vocabulary(ops, L):
    r = np.random.default_rng(0)
    for N in (10, 3000, 20001):
        x = r.standard_normal((4, N)).astype(np.float32)
        t = np.array([1, N, 2 ** 31 - 1, -2 ** 31], np.int32)
        assert status(L) == 0
        logp, ent, stats = ops.token_logprob_fwd(x, t)
        assert status(L) == 8
        assert np.isfinite(logp[0]) and np.all(np.isnan(logp[1:3])) and logp[3] == 0.0 and np.all(stats[1:] == 0.0)
        dx = ops.token_logprob_bwd(x, t, stats, np.ones(4, np.float32))
        assert np.all(dx[1:] == 0.0) and np.all(np.isfinite(dx))
        out = ops.policy_loss(x, t, np.full(4, -2, np.float32), np.ones(4, np.float32))
        assert status(L) == 8
        assert np.isnan(out["loss"]) and out["rows"] == 3 and np.all(out["dlogits"][1:] == 0.0) and np.all(np.isfinite(out["dlogits"]))


def test_every_row_left_out(ops):
    x = np.full((3, 50), np.nan, np.float32)
    t = np.full(3, -1, np.int32)
    bad = np.full(3, np.nan, np.float32)
    out = ops.policy_loss(x, t, bad, bad, bad, kl_coef=0.1, entropy_coef=0.1)
    assert out["loss"] == 0.0 and out["rows"] == 0 and np.all(out["dlogits"] == 0.0) and np.all(out["token_loss"] == 0.0)
    out = ops.policy_loss(x, np.zeros(3, np.int32), bad, bad, bad, np.zeros(3, np.float32), kl_coef=0.1)
    assert out["loss"] == 0.0 and out["rows"] == 0 and np.all(out["dlogits"] == 0.0)


# ------------------------------------------------------------------ layouts
@pytest.mark.parametrize("N,ld,shift,ld_d,shift_d", [(10, 10, 1, 13, 2), (1000, 1003, 3, 1000, 0), (4096, 4100, 0, 4097, 1), (8192, 8192, 1, 8192, 1),
                                                    (8190, 8195, 2, 8190, 3), (20000, 20001, 1, 20004, 0), (50257, 50257, 0, 50260, 3),
                                                    (131071, 131073, 3, 131073, 3)])
def test_strides_and_alignment(ops, L, N, ld, shift, ld_d, shift_d):
    """Rows at every alignment, in buffers whose other floats must stay as they are; in place where the layouts agree."""
    r = np.random.default_rng(N)
    M = 5
    x, t = logits(r, M, N, left=0.2)
    t[0], x[0] = N - 1, 0.5
    lw, ew, _ = ops.token_logprob_fwd(x, t)
    adv, old = r.standard_normal(M).astype(np.float32), (lw - 0.05).astype(np.float32)
    want = ops.policy_loss(x, t, old, adv, entropy_coef=0.1)

    def spread(a, stride, off):
        buf = np.full(off + M * stride + 8, 77.0, np.float32)
        for i in range(M):
            buf[off + i * stride:off + i * stride + N] = a[i]
        return buf

    def gather(buf, stride, off):
        rows = np.stack([buf[off + i * stride:off + i * stride + N] for i in range(M)])
        rest = buf.copy()
        for i in range(M):
            rest[off + i * stride:off + i * stride + N] = 77.0
        assert np.all(rest == 77.0), "floats between the rows were written"
        return rows
    hx = spread(x, ld, shift)
    xb, tb = ops.DevBuf.from_host(hx), ops.DevBuf.from_host(t)
    lp, en, st = ops.DevBuf(M * 4), ops.DevBuf(M * 4), ops.DevBuf(M * 8)
    L.call("znn_token_logprob_fwd", xb.ptr + 4 * shift, ld, tb.ptr, 1.0, lp.ptr, en.ptr, st.ptr, M, N)
    # another alignment deals the columns to other lanes: equal to rounding only
    K = row_k(np.where((t >= 0)[:, None], x, 0.0), 1.0)
    within(lp.to_host((M,)), lw, 2 * K * U + 2 * U * np.abs(lw), "logp")
    ob, ab, loss, tl = ops.DevBuf.from_host(old), ops.DevBuf.from_host(adv), ops.DevBuf(8), ops.DevBuf(M * 4)
    size = np.abs(want["dlogits"]).max()

    def run(dst, stride):
        L.call("znn_policy_loss", xb.ptr + 4 * shift, ld, tb.ptr, 1.0, ob.ptr, None, ab.ptr, None, 0.2, 0.2, 0.0, 0.1, loss.ptr, tl.ptr, None, None,
               dst, stride, M, N)
    db = ops.DevBuf.from_host(spread(np.full((M, N), 5.0, np.float32), ld_d, shift_d))
    run(db.ptr + 4 * shift_d, ld_d)
    got = gather(db.to_host((shift_d + M * ld_d + 8,)), ld_d, shift_d)
    within(got, want["dlogits"], 4 * K.max() * (1 + np.log(N)) * U * size, "dlogits")
    gb, hb = ops.DevBuf.from_host(adv), ops.DevBuf.from_host(old)
    db2 = ops.DevBuf.from_host(spread(np.full((M, N), 5.0, np.float32), ld_d, shift_d))
    L.call("znn_token_logprob_bwd", xb.ptr + 4 * shift, ld, tb.ptr, 1.0, st.ptr, en.ptr, gb.ptr, hb.ptr, db2.ptr + 4 * shift_d, ld_d, 0, M, N)
    apart = gather(db2.to_host((shift_d + M * ld_d + 8,)), ld_d, shift_d)
    # in place over the logits
    keep = ops.DevBuf.from_host(hx)
    L.call("znn_token_logprob_bwd", keep.ptr + 4 * shift, ld, tb.ptr, 1.0, st.ptr, en.ptr, gb.ptr, hb.ptr, keep.ptr + 4 * shift, ld, 0, M, N)
    np.testing.assert_array_equal(gather(keep.to_host((shift + M * ld + 8,)), ld, shift), apart)
    run(xb.ptr + 4 * shift, ld)
    np.testing.assert_array_equal(gather(xb.to_host((shift + M * ld + 8,)), ld, shift), got)


def test_same_bits_every_time(ops):
    r = np.random.default_rng(11)
    x, t = logits(r, 40, 20011)
    adv, old = r.standard_normal(40).astype(np.float32), np.full(40, -3, np.float32)
    a = ops.policy_loss(x, t, old, adv, entropy_coef=0.1)
    for _ in range(3):
        b = ops.policy_loss(x, t, old, adv, entropy_coef=0.1)
        for k in a:
            np.testing.assert_array_equal(a[k], b[k])


def test_rows_beyond_32_bit_offsets(ops, L):
    """More than 2^31 logits: only the last rows are in use, and they are right."""
    N, M = 131072, 16500                                     # 2.16e9 floats, 8.7 GB
    r = np.random.default_rng(1)
    x = r.standard_normal((2, N)).astype(np.float32)
    t = np.full(M, -1, np.int32)
    t[-2:] = [5, N - 1]
    big = ops.DevBuf(M * N * 4)
    L.call("znn_memcpy_h2d", big.ptr + (M - 2) * N * 4, x.ctypes.data, x.nbytes)
    tb = ops.DevBuf.from_host(t)
    lp, st = ops.DevBuf(M * 4), ops.DevBuf(M * 8)
    L.call("znn_token_logprob_fwd", big.ptr, N, tb.ptr, 1.0, lp.ptr, None, st.ptr, M, N)
    got = lp.to_host((M,))
    want = ops.token_logprob_fwd(x, t[-2:])
    within(got[-2:], want[0], (2 * row_k(x, 1.0) + np.abs(want[0])) * U, "logp")   # (see below)
    assert np.all(got[:-2] == 0.0)
    g = np.ones(M, np.float32)
    gb = ops.DevBuf.from_host(g)
    L.call("znn_token_logprob_bwd", big.ptr, N, tb.ptr, 1.0, st.ptr, None, gb.ptr, None, big.ptr, N, 0, M, N)
    tail = np.empty((2, N), np.float32)
    L.call("znn_memcpy_d2h", tail.ctypes.data, big.ptr + (M - 2) * N * 4, tail.nbytes)
    # a call of two rows may deal a row's columns out differently: either sum is good to K u, so the two differ by at most 2 K u, and
    # with them every p_j = exp(d_j) / s, which the gradient is (1 - p_j at the target, where 2 K u p_j <= 2 K u |1 - p_j| + 2 K u p_j)
    again = ops.token_logprob_bwd(x, t[-2:], want[2], g[-2:])
    within(tail, again, 2 * row_k(x, 1.0)[:, None] * U * np.maximum(np.abs(again), np.exp(want[0])[:, None] * (np.arange(N) == t[-2:, None])), "dlogits")


# ------------------------------------------------------------------ preference loss
def ragged(r, P, M, tail=3):
    return np.concatenate([[0], np.sort(r.integers(0, max(M - tail, 0) + 1, 2 * P))]).astype(np.int32)


@pytest.mark.parametrize("P,M", [(1, 1), (1, 0), (1, 2), (2, 7), (4, 163), (8, 1000), (9, 40), (33, 5000), (700, 3001), (3, 100001), (1, 70000), (1025, 9)])
@pytest.mark.parametrize("reference,masked,by_length,smooth,margin", [(True, False, False, 0.0, 0.0), (True, True, True, 0.1, 0.0), (False, True, False, 0.2, 0.5),
                                                                     (False, False, True, 0.0, 0.3)])
def test_preference_loss(ops, P, M, reference, masked, by_length, smooth, margin):
    r = np.random.default_rng(P * 31 + M)
    off = ragged(r, P, M)
    logp = (-3 * r.random(M)).astype(np.float32)
    ref = (logp + 0.3 * r.standard_normal(M)).astype(np.float32) if reference else None
    t = None
    if masked:
        t = np.where(r.random(M) < 0.3, -1, 4).astype(np.int32)
        logp[t < 0] = np.nan
    before = r.standard_normal(M).astype(np.float32)
    beta, smooth, margin = (float(np.float32(v)) for v in (0.3, smooth, margin))
    got = ops.preference_loss(logp, off, ref, t, beta, smooth, margin, by_length, before)
    lz, rz = (np.where(np.isnan(v), 0.0, v) if v is not None else None for v in (logp, ref))
    want = ft.preference(lz, off, rz, t, beta, smooth, margin, by_length, before)
    # everything is summed in fp64: what is left is the rounding of the outputs, and 1e-12 for fp64 sums in another order
    for k in ("pair_loss", "rewards", "dlogp"):
        within(got[k], want[k], U * np.abs(want[k]) * 1.001 + 1e-12, k)
    # the loss is the mean of pair_loss as it was rounded: |mean(l (1 + a)) - mean(l)| <= u mean(l) for |a| <= u and l >= 0, and the
    # mean is rounded once more, u mean(l): together 2 u
    within(got["loss"], want["loss"], 2 * U * want["loss"] * 1.001 + 1e-12, "loss")
    np.testing.assert_array_equal(got["dlogp"][off[-1]:], before[off[-1]:])   # rows behind the last sequence


def test_preference_gradient_is_the_losses_slope(ops):
    """Differences with h = 2^-6: h^2 / 6 times the third derivative (beta^3 / P below 0.1) = 5e-6, loss error 6e-8 / h = 4e-6."""
    r = np.random.default_rng(2)
    off = np.array([0, 3, 5, 9, 10], np.int32)
    logp = np.round(-r.random(12) * 64).astype(np.float32) / 64
    got = ops.preference_loss(logp, off, None, None, 0.5, 0.1, 0.1, True)["dlogp"]
    h = 2.0 ** -6
    for i in range(12):
        a, b = logp.copy(), logp.copy()
        a[i] += h
        b[i] -= h
        d = [float(ops.preference_loss(v, off, None, None, 0.5, 0.1, 0.1, True)["loss"]) for v in (a, b)]
        assert abs((d[0] - d[1]) / (2 * h) - got[i]) < 2e-5


def test_preference_offsets_out_of_order(ops, L):
    """A pair whose offsets leave 0 .. M or descend is reported and touches no row; its neighbours are as ever."""
    logp = np.linspace(-2, -1, 20).astype(np.float32)
    before = np.full(20, 9.0, np.float32)
    for bad in ([0, 3, 6, 5, 8], [0, 3, 6, 9, 21], [0, 3, 6, 2 ** 31 - 1, 10], [0, 3, 6, -5, 10], [0, 3, 6, 9, -1]):
        off = np.array(bad, np.int32)
        assert status(L) == 0
        got = ops.preference_loss(logp, off, dlogp=before)
        assert status(L) == 8
        want = ft.preference(logp, [0, 3, 6], beta=float(np.float32(0.1)))
        within(got["rewards"][:2], want["rewards"], 2 * U, "rewards")
        assert np.isnan(got["loss"]) and np.isnan(got["pair_loss"][1]) and np.all(np.isnan(got["rewards"][2:]))
        assert np.all(got["dlogp"][6:] == 9.0)
    got = ops.preference_loss(logp, np.array([-1, 3, 6], np.int32), dlogp=before)
    assert status(L) == 8 and np.isnan(got["loss"]) and np.all(got["dlogp"] == 9.0)


def test_preference_extreme_margins(ops):
    """Margins of +-1000: the loss is 0 or the margin itself, the slope 0 or 1, nothing overflows."""
    logp = np.array([0.0, -1000.0, -1000.0, 0.0], np.float32)
    got = ops.preference_loss(logp, np.array([0, 1, 2, 3, 4], np.int32), beta=1.0)
    np.testing.assert_array_equal(got["pair_loss"], np.array([0.0, 1000.0], np.float32))
    np.testing.assert_array_equal(got["dlogp"], np.array([0.0, 0.0, -0.5, 0.5], np.float32))


# ------------------------------------------------------------------ gradient norm, clipping, clipped steps
SETS = [[1], [3, 0, 5], [100352, 128, 8192, 64, 640, 10], [1 << 20], [(1 << 20) + 3], [3000001], [7] * 40, [8191, 8192, 8193] * 5, [5] * 2500, [70000] * 30, [0, 0]]


@pytest.mark.parametrize("sizes", SETS, ids=lambda s: f"{len(s)}x{s[0]}")
@pytest.mark.parametrize("scale,max_norm", [(1.0, np.inf), (0.125, 1e-3), (-2.0, 1e9)])
def test_grad_norm_and_clip(ops, sizes, scale, max_norm):
    r = np.random.default_rng(len(sizes) + sizes[0])
    grads = [(r.standard_normal(n) * 10 ** r.uniform(-3, 1)).astype(np.float32) for n in sizes]
    max_norm = float(np.float32(max_norm))
    want = ft.grad_norm(grads, max_norm, scale)
    got = ops.grad_norm(grads, max_norm, scale)
    within(got, want, 1.001 * U * np.array(want), "norm and factor")     # fp64 inside, one rounding each
    after = [g.copy() for g in grads]
    both = ops.clip_grads(after, max_norm, scale)
    np.testing.assert_array_equal(both, got)
    for a, g in zip(after, grads):
        np.testing.assert_array_equal(a, g if got[1] == 1.0 else g * got[1])


def test_grad_norm_at_every_alignment(ops, L):
    """Tensors that lie one after the other at any multiple of 4 bytes; what lies between them is not counted or scaled."""
    r = np.random.default_rng(3)
    for total in (300, 40000, 2000000):
        host = r.standard_normal(total + 64).astype(np.float32)
        cuts = np.sort(r.integers(0, total, 10))
        spans = [(int(a) + k % 4, int(b)) for k, (a, b) in enumerate(zip(cuts[:-1], cuts[1:])) if b > a + 3]
        buf, res = ops.DevBuf.from_host(host), ops.DevBuf(ops.GRAD_NORM_FLOATS * 4)
        ptrs = (C.c_void_p * len(spans))(*[buf.ptr + 4 * a for a, _ in spans])
        counts = (C.c_size_t * len(spans))(*[b - a for a, b in spans])
        L.call("znn_grad_norm", ptrs, counts, len(spans), 1.0, 0.5, res.ptr)
        norm, factor = res.to_host((2,))
        want = ft.grad_norm([host[a:b] for a, b in spans], 0.5)
        within([norm, factor], want, 1.001 * U * np.array(want), "norm and factor")
        L.call("znn_clip_grads", ptrs, counts, len(spans), res.ptr)
        expect = host.copy()
        for a, b in spans:
            expect[a:b] *= factor
        np.testing.assert_array_equal(buf.to_host(host.shape), expect)


@pytest.mark.parametrize("n", [5, 5000, 2000003])
def test_grad_norm_range(ops, n):
    """No finite gradients overflow or vanish: 3e38 and 1e-40 (below the type's normal range)"""
    for value in (3e38, 1e-40):
        g = np.zeros(n, np.float32)
        g[[0, n // 2, n - 1]] = value
        norm = float(np.float32(value)) * np.sqrt(3.0)
        got = ops.grad_norm([g], 1.0, 0.25)
        want = 0.25 * norm
        if value > 1:
            within(got, (want, 1.0 / want), (U * want, max(U / want, 2.0 ** -150)), "norm")
        else:
            within(got, (want, 1.0), (2.0 ** -150, 0.0), "norm")
    for poison in (np.nan, np.inf, -np.inf):
        g = np.ones(n, np.float32)
        g[n - 1] = poison
        keep = g.copy()
        norm, factor = ops.clip_grads([g], 1.0)
        assert not np.isfinite(norm) and factor == 0.0
        np.testing.assert_array_equal(g, keep)
        w, m, v = (np.full(n, 0.5, np.float32) for _ in range(3))
        ops.adam_step_clipped(w, g, m, v, 1e-3, 0.9, 0.99, 1e-8, 1.0, 1.0)
        ops.sgd_step_clipped(w, g, v, 1e-3, 0.9, 1.0)
        assert np.all(w == 0.5) and np.all(m == 0.5) and np.all(v == 0.5)


@pytest.mark.parametrize("n", [1, 6, 1024, 109386, 1 << 20, 1048579])
@pytest.mark.parametrize("clipped,scale", [(False, 1.0), (True, 1.0), (True, 0.125)])
def test_clipped_steps(ops, n, clipped, scale):
    """Bit for bit the unclipped step on a gradient that was multiplied by the factor beforehand."""
    r = np.random.default_rng(n)
    w, g, m = (r.standard_normal(n).astype(np.float32) for _ in range(3))
    v = r.random(n).astype(np.float32)
    max_norm = 0.25 * float(np.linalg.norm(g)) * scale if clipped else np.inf
    for t in (1.0, 7.0):
        a, b = [x.copy() for x in (w, m, v)], [x.copy() for x in (w, m, v)]
        norm, factor = ops.adam_step_clipped(a[0], g, a[1], a[2], 1e-2, 0.9, 0.95, 1e-6, t, max_norm, scale)
        assert (factor < 1.0) == clipped
        ops.adam_step(b[0], g * np.float32(np.float32(scale) * factor), b[1], b[2], 1e-2, 0.9, 0.95, 1e-6, t)
        for x, y in zip(a, b):
            np.testing.assert_array_equal(x, y)
    for momentum in (0.0, 0.9):
        a, b = [w.copy(), v.copy()], [w.copy(), v.copy()]
        ops.sgd_step_clipped(a[0], g, a[1] if momentum else None, 0.1, momentum, max_norm, scale)
        ops.sgd_step(b[0], g * np.float32(np.float32(scale) * factor), b[1] if momentum else None, 0.1, momentum)
        for x, y in zip(a, b):
            np.testing.assert_array_equal(x, y)


def test_clipped_steps_unaligned(ops, L):
    """w, g, m, v at alignments of their own"""
    r = np.random.default_rng(8)
    n = 40003
    host = [r.random(n + 4).astype(np.float32) for _ in range(4)]
    res = ops.DevBuf.from_host(np.array([2.0, 0.5, 0.0, 0.0], np.float32))
    for shifts in ((0, 0, 0, 0), (1, 1, 1, 1), (0, 1, 2, 3), (3, 0, 0, 2)):
        bufs = [ops.DevBuf.from_host(h) for h in host]
        p = [b.ptr + 4 * s for b, s in zip(bufs, shifts)]
        L.call("znn_adam_step_clipped", p[0], p[1], p[2], p[3], 1e-2, 0.9, 0.95, 1e-6, 3.0, 1.0, res.ptr, n)
        w, g, m, v = (h[s:s + n].copy() for h, s in zip(host, shifts))
        ops.adam_step(w, g * np.float32(0.5), m, v, 1e-2, 0.9, 0.95, 1e-6, 3.0)
        for b, s, h, x in zip(bufs, shifts, host, (w, g, m, v)):
            out = b.to_host(h.shape)
            np.testing.assert_array_equal(out[s:s + n], x)
            np.testing.assert_array_equal(out[:s], h[:s])
            np.testing.assert_array_equal(out[s + n:], h[s + n:])


# ------------------------------------------------------------------ streams, capture, the calls in a row
def test_a_run_of_them_on_another_stream_and_captured(ops, L):
    """Scoring, preference loss, its gradient, clipping and an Adam step, as a training step has them: eager on the shim's
    stream, eager on another stream, and captured there into a graph that is replayed twice; two graphs with buffers of
    their own run at the same time."""
    torch = pytest.importorskip("torch")
    M, N, P = 60, 5003, 4

    class Step:
        def __init__(self, seed):
            r = np.random.default_rng(seed)
            x, t = logits(r, M, N, left=0.2)
            off = ragged(r, P, M)
            up = ops.DevBuf.from_host
            self.x, self.t, self.off = up(np.nan_to_num(x, nan=0.0)), up(t), up(off)
            self.ref = up((-8 + r.standard_normal(M)).astype(np.float32))
            self.lp, self.st, self.dlp = ops.DevBuf(M * 4), ops.DevBuf(M * 8), up(np.zeros(M, np.float32))
            self.loss, self.pl, self.rw = ops.DevBuf(4), ops.DevBuf(P * 4), ops.DevBuf(8 * P)
            self.dx, self.res = ops.DevBuf(M * N * 4), ops.DevBuf(ops.GRAD_NORM_FLOATS * 4)
            self.w0 = r.standard_normal(M * N).astype(np.float32)
            self.w, self.m, self.v = up(self.w0), up(np.zeros(M * N, np.float32)), up(np.zeros(M * N, np.float32))
            self.ptrs, self.counts = (C.c_void_p * 1)(self.dx.ptr), (C.c_size_t * 1)(M * N)

        def run(self):
            L.call("znn_token_logprob_fwd", self.x.ptr, N, self.t.ptr, 1.0, self.lp.ptr, None, self.st.ptr, M, N)
            L.call("znn_preference_loss", self.lp.ptr, self.ref.ptr, self.t.ptr, self.off.ptr, 0.1, 0.0, 0.0, 0, self.loss.ptr, self.pl.ptr, self.rw.ptr,
                   self.dlp.ptr, P, M)
            L.call("znn_token_logprob_bwd", self.x.ptr, N, self.t.ptr, 1.0, self.st.ptr, None, self.dlp.ptr, None, self.dx.ptr, N, 0, M, N)
            L.call("znn_grad_norm", self.ptrs, self.counts, 1, 1.0, 0.01, self.res.ptr)
            L.call("znn_adam_step_clipped", self.w.ptr, self.dx.ptr, self.m.ptr, self.v.ptr, 1e-2, 0.9, 0.95, 1e-8, 1.0, 1.0, self.res.ptr, M * N)

        def out(self):
            return [self.loss.to_host((1,)), self.dx.to_host((M, N)), self.w.to_host((M * N,)), self.res.to_host((2,))]

    want = []
    for seed in (1, 2):
        s = Step(seed)
        s.run()
        first = s.out()
        s.run()
        want.append((first, s.out()))
    lw = ft.rows(np.nan_to_num(logits(np.random.default_rng(1), M, N, left=0.2)[0], nan=0.0), logits(np.random.default_rng(1), M, N, left=0.2)[1])[0]
    assert np.all(np.isfinite(lw)) and want[0][0][3][1] <= 1.0
    streams = [torch.cuda.Stream() for _ in range(2)]
    steps = [Step(1), Step(2)]
    try:
        for s, st in zip(steps, streams):
            L.call("znn_sync")
            L.call("znn_set_stream", st.cuda_stream)
            s.run()
        for s, st, w in zip(steps, streams, want):
            L.call("znn_set_stream", st.cuda_stream)
            for a, b in zip(s.out(), w[0]):
                np.testing.assert_array_equal(a, b)
        graphs, steps = [], [Step(1), Step(2)]
        torch.cuda.synchronize()
        for s, st in zip(steps, streams):
            L.call("znn_set_stream", st.cuda_stream)
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=st, capture_error_mode="thread_local"):
                s.run()
            graphs.append(g)
        for _ in range(2):
            for g, st in zip(graphs, streams):
                with torch.cuda.stream(st):
                    g.replay()
        torch.cuda.synchronize()
        for s, w in zip(steps, want):
            for a, b in zip(s.out(), w[1]):
                np.testing.assert_array_equal(a, b)
    finally:
        L.call("znn_set_stream", None)


@pytest.mark.parametrize("M,N", [(61, 700), (700, 40), (600, 9001), (20, 40000)])
def test_policy_loss_captured_and_on_two_streams(ops, L, M, N):
    """Two policy losses with buffers of their own, captured on two streams and replayed at the same time, and eager ones that follow
    one another without a wait while the inputs change in between: every result is the one of a call alone."""
    torch = pytest.importorskip("torch")

    class Call:
        def __init__(self, seed):
            r = np.random.default_rng(seed)
            self.r = r
            self.host = []
            for _ in range(3):
                x, t = logits(r, M, N)
                self.host.append((np.nan_to_num(x, nan=0.0, neginf=-np.inf), t))
            self.old, self.adv = np.full(M, -4, np.float32), r.standard_normal(M).astype(np.float32)
            up = ops.DevBuf.from_host
            self.xs = [up(h[0]) for h in self.host]
            self.ts = [up(h[1]) for h in self.host]
            self.x, self.t, self.o, self.a = ops.DevBuf(4 * M * N), ops.DevBuf(4 * M), up(self.old), up(self.adv)
            self.loss, self.tl, self.lp, self.dx = ops.DevBuf(8), ops.DevBuf(4 * M), ops.DevBuf(4 * M), ops.DevBuf(4 * M * N)
            self.keep = [[ops.DevBuf(8), ops.DevBuf(4 * M * N)] for _ in range(3)]

        def load(self, k):
            L.call("znn_memcpy_d2d", self.x.ptr, self.xs[k].ptr, 4 * M * N)
            L.call("znn_memcpy_d2d", self.t.ptr, self.ts[k].ptr, 4 * M)

        def run(self):
            L.call("znn_policy_loss", self.x.ptr, N, self.t.ptr, 1.0, self.o.ptr, None, self.a.ptr, None, 0.2, 0.2, 0.0, 0.0, self.loss.ptr,
                   self.tl.ptr, self.lp.ptr, None, self.dx.ptr, N, M, N)

        def save(self, k):
            L.call("znn_memcpy_d2d", self.keep[k][0].ptr, self.loss.ptr, 8)
            L.call("znn_memcpy_d2d", self.keep[k][1].ptr, self.dx.ptr, 4 * M * N)

        def check(self, k):
            want = ops.policy_loss(*self.host[k], self.old, self.adv)
            got = self.keep[k][0].to_host((2,))
            assert got[0] == want["loss"] and got[1] == want["rows"]
            np.testing.assert_array_equal(self.keep[k][1].to_host((M, N)), want["dlogits"])
    calls, streams, graphs = [Call(1), Call(2)], [torch.cuda.Stream() for _ in range(2)], []
    torch.cuda.synchronize()
    try:
        for k in range(3):
            for c, st in zip(calls, streams):
                L.call("znn_set_stream", st.cuda_stream)
                c.load(k)
                c.run()
                c.save(k)
        torch.cuda.synchronize()
        L.call("znn_set_stream", None)
        for c in calls:
            for k in range(3):
                c.check(k)
        for c, st in zip(calls, streams):
            L.call("znn_set_stream", st.cuda_stream)
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=st, capture_error_mode="thread_local"):
                c.run()
            graphs.append(g)
        for k in (2, 0, 1):
            for c, st, g in zip(calls, streams, graphs):
                L.call("znn_set_stream", st.cuda_stream)
                c.load(k)
                with torch.cuda.stream(st):
                    g.replay()
                c.save(k)
        torch.cuda.synchronize()
    finally:
        L.call("znn_set_stream", None)
    for c in calls:
        for k in range(3):
            c.check(k)


@pytest.mark.parametrize("M,N", [(30, 700), (600, 1300), (520, 9001)])
def test_calls_behind_copies_and_a_join_captured(ops, L, M, N):
    """A graph whose logits come from a copy on one stream and whose targets come from another stream, joined right before the
    policy loss, with a norm of the gradient on the second stream behind it: three replays with other inputs."""
    torch = pytest.importorskip("torch")
    r = np.random.default_rng(M)
    up = ops.DevBuf.from_host
    sets = []
    for _ in range(3):
        x, t = logits(r, M, N)
        sets.append((np.nan_to_num(x, nan=0.0, neginf=-np.inf), t))
    old, adv = np.full(M, -4, np.float32), r.standard_normal(M).astype(np.float32)
    want = [ops.policy_loss(x, t, old, adv) for x, t in sets]
    o, a = up(old), up(adv)
    x0, t0, x, t = ops.DevBuf(4 * M * N), ops.DevBuf(4 * M), ops.DevBuf(4 * M * N), ops.DevBuf(4 * M)
    loss, tl, dx, res = ops.DevBuf(8), ops.DevBuf(4 * M), ops.DevBuf(4 * M * N), ops.DevBuf(ops.GRAD_NORM_FLOATS * 4)
    ptrs, counts = (C.c_void_p * 1)(dx.ptr), (C.c_size_t * 1)(M * N)
    main, side = torch.cuda.Stream(), torch.cuda.Stream()
    L.call("znn_sync")
    g = torch.cuda.CUDAGraph()
    try:
        with torch.cuda.graph(g, stream=main, capture_error_mode="thread_local"):
            side.wait_stream(main)
            L.call("znn_set_stream", side.cuda_stream)
            L.call("znn_memcpy_d2d", t.ptr, t0.ptr, 4 * M)
            L.call("znn_set_stream", main.cuda_stream)
            L.call("znn_memcpy_d2d", x.ptr, x0.ptr, 4 * M * N)
            main.wait_stream(side)
            L.call("znn_policy_loss", x.ptr, N, t.ptr, 1.0, o.ptr, None, a.ptr, None, 0.2, 0.2, 0.0, 0.0, loss.ptr, tl.ptr, None, None, dx.ptr, N, M, N)
            side.wait_stream(main)
            L.call("znn_set_stream", side.cuda_stream)
            L.call("znn_grad_norm", ptrs, counts, 1, 1.0, 0.5, res.ptr)
            main.wait_stream(side)
            L.call("znn_set_stream", main.cuda_stream)
            L.call("znn_clip_grads", ptrs, counts, 1, res.ptr)
        for (hx, ht), w in zip(sets, want):
            bx, bt = up(hx), up(ht)
            L.call("znn_memcpy_d2d", x0.ptr, bx.ptr, 4 * M * N)
            L.call("znn_memcpy_d2d", t0.ptr, bt.ptr, 4 * M)
            with torch.cuda.stream(main):
                g.replay()
            L.call("znn_sync")
            got = loss.to_host((2,))
            assert got[0] == w["loss"] and got[1] == w["rows"]
            factor = res.to_host((2,))[1]
            assert 0 < factor <= 1
            np.testing.assert_array_equal(dx.to_host((M, N)), w["dlogits"] * factor)
    finally:
        L.call("znn_set_stream", None)


@pytest.mark.parametrize("M,N", [(40, 40001), (24, 131072)])
def test_policy_gradient_over_the_logits_of_rows_in_parts(ops, L, M, N):
    """In place where the blocks of a cluster share a row: whichever of them writes first, the others have the target's logit."""
    r = np.random.default_rng(N)
    up = ops.DevBuf.from_host
    x, t = logits(r, M, N)
    x = np.nan_to_num(x, nan=0.0, neginf=-np.inf)
    old, adv = np.full(M, -4, np.float32), r.standard_normal(M).astype(np.float32)
    want = ops.policy_loss(x, t, old, adv)
    bt, o, a, loss, tl = up(t), up(old), up(adv), ops.DevBuf(8), ops.DevBuf(4 * M)
    for _ in range(20):
        b = up(x)
        L.call("znn_policy_loss", b.ptr, N, bt.ptr, 1.0, o.ptr, None, a.ptr, None, 0.2, 0.2, 0.0, 0.0, loss.ptr, tl.ptr, None, None, b.ptr, N, M, N)
        assert loss.to_host((2,))[0] == want["loss"]
        np.testing.assert_array_equal(b.to_host((M, N)), want["dlogits"])


def test_tensors_that_overlap_are_not_clipped(ops, L):
    host = np.arange(64, dtype=np.float32)
    b, res = ops.DevBuf.from_host(host), ops.DevBuf(ops.GRAD_NORM_FLOATS * 4)
    twice = (C.c_void_p * 2)(b.ptr, b.ptr + 4 * 31)
    counts = (C.c_size_t * 2)(32, 33)
    L.call("znn_grad_norm", twice, counts, 2, 1.0, 1.0, res.ptr)   # a float of both counts twice
    want = np.sqrt(np.square(host.astype(np.float64)).sum() + 31.0 ** 2)
    assert abs(float(res.to_host((2,))[0]) - want) <= want * np.finfo(np.float32).eps
    with pytest.raises(Exception, match="overlap"):
        L.call("znn_clip_grads", twice, counts, 2, res.ptr)
    np.testing.assert_array_equal(b.to_host((64,)), host)
    counts = (C.c_size_t * 2)(31, 33)
    L.call("znn_clip_grads", twice, counts, 2, res.ptr)
    factor = res.to_host((2,))[1]
    np.testing.assert_array_equal(b.to_host((64,)), host * factor)


@pytest.mark.parametrize("N", [1, 3, 31, 32, 33, 64, 65, 127, 128, 129, 256, 257, 511, 512, 513, 1023, 1024])
@pytest.mark.parametrize("M,pad,shift,ce", [(1, 0, 0, 0.0), (3, 0, 0, 0.1), (131, 0, 0, 0.0), (130, 3, 1, 0.1), (67, 4, 0, 0.0)])
def test_short_rows_together_and_alone(ops, L, N, M, pad, shift, ce):
    """A short row gives the same bits among others as alone (where groups of lanes take several rows), beside rows that are left out and
    hold NaN and rows with a bad target, in place, and floats between the rows and behind the last one stay."""
    r = np.random.default_rng(N * 7 + M)
    x, t = logits(r, M, N, left=0.3)
    t[r.random(M) < 0.05] = N
    x[t < 0] = np.nan
    ld = N + pad
    old, adv = np.full(M, -3, np.float32), r.standard_normal(M).astype(np.float32)
    w = r.random(M).astype(np.float32) + 0.5
    w[r.random(M) < 0.1] = 0
    buf = np.full(shift + M * ld + 64, 77.0, np.float32)
    for i in range(M):
        buf[shift + i * ld:shift + i * ld + N] = x[i]
    up = ops.DevBuf.from_host
    tb, ob, ab, wb = up(t), up(old), up(adv), up(w)
    loss, tl, lp, en = ops.DevBuf(8), up(np.full(M + 8, 5, np.float32)), up(np.full(M + 8, 5, np.float32)), up(np.full(M + 8, 5, np.float32))

    def run(b, first, rows):
        at = b.ptr + 4 * (shift + first * ld)
        L.call("znn_policy_loss", at, ld, tb.ptr + 4 * first, 1.0, ob.ptr + 4 * first, None, ab.ptr + 4 * first, wb.ptr + 4 * first, 0.2, 0.2, 0.0, ce,
               loss.ptr, tl.ptr + 4 * first, lp.ptr + 4 * first, en.ptr + 4 * first, at, ld, rows, N)
    together, alone = up(buf), up(buf)
    run(together, 0, M)
    a = [together.to_host(buf.shape)] + [v.to_host((M + 8,)) for v in (tl, lp, en)]
    for i in range(M):
        run(alone, i, 1)
    b = [alone.to_host(buf.shape)] + [v.to_host((M + 8,)) for v in (tl, lp, en)]
    for p, q in zip(a, b):
        np.testing.assert_array_equal(p, q)
    rest = a[0].copy()
    for i in range(M):
        row = rest[shift + i * ld:shift + i * ld + N]
        assert np.all(np.isfinite(row)) and (0 <= t[i] < N and w[i] != 0 or np.all(row == 0.0))
        row[:] = 77.0
    assert np.all(rest == 77.0) and all(np.all(v[M:] == 5.0) for v in a[1:])
    want = ft.policy(np.where((t < 0)[:, None], 0.0, x), t, old, adv, weights=w, ce=ce)
    within(a[2][:M], want["logp"], 4 * (row_k(np.where((t >= 0)[:, None], np.nan_to_num(x, nan=0.0, neginf=0.0), 0.0), 1.0) + np.abs(np.nan_to_num(want["logp"]))) * U, "logp")
    status(L)


@pytest.mark.parametrize("M,N", [(450, 1100), (520, 1501), (450, 2000), (451, 2100), (450, 2816), (300, 2900), (450, 2900), (520, 4100), (450, 4999), (450, 5121),
                                 (447, 6000), (450, 8191), (300, 9001), (450, 9001), (520, 12288), (450, 12500), (446, 26000), (300, 51300), (450, 51300)])
def test_many_rows_of_every_length(ops, M, N):
    """As many rows as take the kernels for large calls: every block size and number of quads that a length asks for."""
    test_token_logprob(ops, M, N, 0.7)
    test_token_logprob_grad(ops, M, N, True, M % 2 == 0)
    test_token_logprob_grad(ops, M, N, False, M % 2 == 1)
    test_policy_loss(ops, M, N, 0.1, 0.02, True, 0.7)
    test_policy_loss(ops, M, N, 0.05, 0.0, False, 1.25)
