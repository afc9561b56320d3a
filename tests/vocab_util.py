"""Inputs and tolerances of the vocabulary tests.

Tolerances are derived, not fitted.  One step of fp32 is 2^-24 of the value.  In units of log 2 an exponent e = y log2(e) carries three
roundings (difference, scale, factor), 3 |e| 2^-24; exp2 by the special-function unit is good to 2^-22.  A row's sum L adds its terms in
chains of at most `chain` additions, a step each.  So with E1 = sum p |e|, E2 = sum p e^2:

    L, relative          rL = 2^-22 + 3 E1 2^-24 + chain 2^-24
    log p of an entry    3 |y| 2^-24 + rL + (|y| + |log L|) 2^-23
    entropy              rL + |log L| 2^-23 + ln 2 (E1 (2^-22 + (chain + 8) 2^-24 + rL) + 3 E2 2^-24)

A gradient p (c0 + c1 log p) takes the relative error of p (that of L, its own exponent and exp2) on each of the two terms, the entropy's
error times p h / t, and half a step of its type on the result; below the normal range half a step is absolute."""
import numpy as np

LN2 = float(np.log(2.0))
HALF_STEP = {"f32": 2.0 ** -24, "bf16": 2.0 ** -8, "f16": 2.0 ** -11}       # relative
SUBNORMAL = {"f32": 2.0 ** -126, "bf16": 2.0 ** -126, "f16": 2.0 ** -25}    # results below the normal range; fp32 and bf16 may be flushed


def row_errors(oracle, X, tau):
    """(log p, p, H, y, rL, tolerance of H) per row; rows without any probability have no error."""
    logp, p, H = oracle.vocab_stats_ref(X, tau)
    M = X.shape[1]
    mx = X.max(1, keepdims=True)
    y = np.where(np.isneginf(X), 0.0, (np.where(np.isneginf(X), 0.0, X) - np.where(np.isneginf(mx), 0.0, mx)) / tau)
    e = np.abs(y) / LN2
    E1, E2 = (p * e).sum(1), (p * e * e).sum(1)
    chain = 64 + M / 256
    rL = 2.0 ** -22 + 3 * E1 * 2.0 ** -24 + chain * 2.0 ** -24
    logL = np.where(np.isneginf(mx[:, 0]), 0.0, -logp.max(1))
    tH = rL + np.abs(logL) * 2.0 ** -23 + LN2 * (E1 * (2.0 ** -22 + (chain + 8) * 2.0 ** -24 + rL) + 3 * E2 * 2.0 ** -24)
    return logp, p, H, y, rL, tH


def logp_tolerance(y, rL, logp):
    """of entries with exponent y (per row or per row and entry)."""
    rL = rL.reshape(rL.shape + (1,) * (y.ndim - rL.ndim))
    logL = np.abs(np.where(np.isfinite(logp), y - np.where(np.isfinite(logp), logp, 0.0), 0.0))
    return 3 * np.abs(y) * 2.0 ** -24 + rL + (np.abs(y) + logL) * 2.0 ** -23


def close(got, ref, tol, what):
    """Equal where the reference is infinite or NaN, within `tol` elsewhere; a reference beyond fp32's range is infinite."""
    got = np.asarray(got, dtype=np.float64)
    with np.errstate(invalid="ignore"):
        ref = np.where(np.abs(ref) > float(np.finfo(np.float32).max), np.sign(ref) * np.inf, ref)
    assert got.shape == ref.shape, f"{what}: shape {got.shape}, expected {ref.shape}"
    fine = np.isfinite(ref)
    assert np.array_equal(np.isnan(got), np.isnan(ref)), f"{what}: NaN in other places"
    odd = ~fine & ~np.isnan(ref)
    assert np.array_equal(got[odd], ref[odd]), f"{what}: infinities differ"
    assert np.isfinite(got[fine]).all(), f"{what}: not finite"
    over = np.abs(got[fine] - ref[fine]) - np.broadcast_to(tol, ref.shape)[fine]
    if over.size:
        k = int(np.argmax(over))
        assert over[k] <= 0, f"{what}: {got[fine][k]!r} for {ref[fine][k]!r}, {over[k]:.3e} beyond the tolerance"


def logprob_grad_tolerance(oracle, X, g, h, hot, tau, dt, ref):
    logp, p, H, y, rL, tH = row_errors(oracle, X, tau)
    lp = np.where(p > 0, logp, 0.0)
    rp = rL[:, None] + 2.0 ** -22 + 3 * np.abs(y) / LN2 * 2.0 ** -24 + 4 * 2.0 ** -24
    g, h = np.abs(g)[:, None], np.abs(h)[:, None]
    size = p * (g + h * (np.abs(lp) + H[:, None]))
    t = size * (rp + 8 * 2.0 ** -24) + p * h * (tH[:, None] + 3 * np.abs(y) * 2.0 ** -24 + np.abs(lp) * 2.0 ** -22) + hot * g * 2.0 ** -22
    return t / tau + np.abs(ref) * HALF_STEP[dt] * (1 + 1e-6) + SUBNORMAL[dt]


def teacher_tolerance(z, p, K):
    """relative error of p_k = exp(z_k - normaliser): the quotient, the difference, expf (2 steps) and the sum of K terms."""
    with np.errstate(invalid="ignore"):
        zz = np.where(p > 0, np.abs(np.where(np.isfinite(z), z, 0.0)), 0.0)
    return (2 * zz.max(1, initial=0.0, keepdims=True) + 2 * zz + 8 + K) * 2.0 ** -23
