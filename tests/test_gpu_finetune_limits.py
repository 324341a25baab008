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
