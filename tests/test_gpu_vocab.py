"""GPU: log probabilities of tokens with entropy and alternatives, and distillation from a teacher's top logits, forward, backward and
in one launch, against the oracle in 64 bits.  Tolerances are derived in vocab_util.py."""
import threading
from concurrent.futures import ThreadPoolExecutor

import numpy as np
import pytest
import torch

from gpu_util import TORCH_DT, back
from vocab_util import HALF_STEP, SUBNORMAL, close, logp_tolerance, logprob_grad_tolerance, row_errors, teacher_tolerance

pytestmark = pytest.mark.gpu

SIZES = [(1, 1), (3, 2), (5, 7), (4, 8), (9, 9), (33, 127), (2, 1000), (200, 1024), (17, 4097), (1, 32768), (3, 40001), (7, 65536),
         (40, 131072), (160, 33333), (2, 262149), (1, 1000003)]


def logits(rng, N, M, dt, *, pad=0, kind="normal"):
    """(device logits, their values in 64 bits, the whole buffer)."""
    x = rng.standard_normal((N, M)) * 3 - np.log1p(np.arange(M) * 8.0 / M)
    lowest = float(torch.finfo(TORCH_DT[dt]).min)
    if kind == "masked":            # most entries -Inf, a row of nothing else, a row with one entry
        x[rng.random((N, M)) < 0.9] = -np.inf
        x[0] = -np.inf
        x[N // 2] = -np.inf
        x[N // 2, M // 3] = 1.5
    elif kind == "lowest":          # masks of the type's lowest value; a row of nothing else is uniform
        x[rng.random((N, M)) < 0.5] = lowest
        x[0] = lowest
    elif kind == "ties":
        x = np.round(x / 4) * 4
        x[N // 2] = 0.0
    elif kind == "rising":          # every element beats all before it
        x = np.broadcast_to(np.linspace(-60, 60, M), (N, M)).copy()
    elif kind == "stripes":         # what is large sits in the shares of few threads: packets 0 to 59 of every 256
        vec = 4 if dt == "f32" else 8
        x += np.where(np.arange(M) // vec % 256 < 60, 30.0, 0.0)
    elif kind == "large":           # far from zero: only differences matter
        x = x + 3e4 if dt == "f16" else x + 1e6
    buf = torch.full((N, M + pad), 7.0, dtype=TORCH_DT[dt], device="cuda")
    buf[:, :M] = torch.from_numpy(x).to(TORCH_DT[dt]).cuda()
    X = buf[:, :M]
    return X, back(X), buf


def dev(a, dtype=torch.float32):
    return torch.from_numpy(np.ascontiguousarray(a)).to(dtype).cuda()


def like(X):
    return torch.full((X.shape[0], max(X.stride(0), X.shape[1])), 7.0, dtype=X.dtype, device="cuda")[:, :X.shape[1]]


def check_score(tylo, oracle, X, X64, targets, tau, K, what):
    N, M = X64.shape
    cp = tylo.allocate_checkpoints_token_logprobs(X)
    got = tylo.token_logprobs(X, dev(targets, torch.int32), temperature=tau, entropy=True, top=K, checkpoints=cp)
    rl, rH = oracle.token_logprobs_ref(X64, targets, tau)
    logp, p, _, y, rL, tH = row_errors(oracle, X64, tau)
    has = (targets >= 0) & (targets < M)
    at = np.where(has, targets, 0)
    rows = np.arange(N)
    close(back(got.logp), rl, np.where(has, logp_tolerance(y[rows, at], rL, logp[rows, at]), 0.0), what + " logp")
    close(back(got.entropy), rH, tH, what + " entropy")
    if K:
        index = oracle.top_alternatives_ref(X64, K)
        assert np.array_equal(back(got.top.index), index), what + " top index"
        take = lambda a: np.take_along_axis(a, index, axis=1)
        close(back(got.top.logp), take(logp), logp_tolerance(take(y), rL, take(logp)), what + " top logp")
    close(back(cp.M), X64.max(1), 0.0, what + " M")
    return got, cp


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("N,M", SIZES)
def test_scores(tylo, oracle, N, M, dt):
    rng = np.random.default_rng(N * 7 + M)
    X, X64, _ = logits(rng, N, M, dt)
    targets = rng.integers(0, M, N)
    for K in sorted({0, 1, min(20, M), min(128, M)}):
        check_score(tylo, oracle, X, X64, targets, 1.0, K, f"top {K}")


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("kind", ["masked", "lowest", "ties", "rising", "stripes", "large"])
@pytest.mark.parametrize("N,M,K,tau", [(5, 300, 256, 1.0), (3, 5000, 256, 0.6), (4, 33001, 64, 2.0), (200, 20011, 100, 1.0), (300, 40000, 64, 1.0),
                                       (300, 10000, 256, 1.0), (2, 200000, 256, 1.0)])
def test_scores_of_odd_rows(tylo, oracle, N, M, K, tau, kind, dt):
    rng = np.random.default_rng(M + K)
    X, X64, _ = logits(rng, N, M, dt, kind=kind, pad=3)
    targets = rng.integers(0, M, N)
    targets[-1] = -1
    if N > 2:
        targets[1] = M
    check_score(tylo, oracle, X, X64, targets, tau, K, kind)


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("M", [9, 1000, 33001, 140000])
def test_nan_and_infinity_reach_their_row_alone(tylo, oracle, M, dt):
    rng = np.random.default_rng(M)
    X, X64, buf = logits(rng, 6, M, dt, pad=5)
    X[1, M // 2] = float("nan")
    X[2, M - 1] = float("inf")
    X[3, 0] = float("nan")
    X[4] = float("-inf")
    X[4, M // 3] = float("nan")
    X64 = back(X)
    K = min(M, 8)
    got = tylo.token_logprobs(X, dev(np.zeros(6), torch.int32), entropy=True, top=K)
    assert np.array_equal(back(got.top.index), oracle.top_alternatives_ref(X64, K))
    bad = np.array([False, True, True, True, True, False])
    for t in (got.logp, got.entropy, got.top.logp[:, 0]):
        assert np.array_equal(np.isnan(back(t)), bad)
    w = torch.ones(6, device="cuda")
    dX, loss = like(X), torch.empty(6, device="cuda")
    tylo.token_logprobs_with_grad_(tylo.Duplicated(loss, w), tylo.Duplicated(X, dX), dev(np.zeros(6), torch.int32))
    assert np.array_equal(np.isnan(back(dX)).all(1), bad) and np.array_equal(np.isnan(back(dX)).any(1), bad)


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("N,M,pad,tau,kind", [(1, 1, 0, 1.0, "normal"), (6, 9, 0, 1.0, "normal"), (5, 1003, 2, 0.6, "masked"), (3, 33001, 0, 2.0, "normal"),
                                              (40, 4096, 8, 1.0, "lowest"), (200, 10007, 0, 0.8, "masked"), (2, 262149, 3, 1.0, "large"), (300, 32768, 0, 1.0, "normal")])
def test_logprob_gradients(tylo, oracle, N, M, pad, tau, kind, dt):
    rng = np.random.default_rng(N + M)
    X, X64, _ = logits(rng, N, M, dt, pad=pad, kind=kind)
    targets = rng.integers(0, M, N)
    if N > 2:
        targets[1], targets[2] = -100, M
    g, h = rng.standard_normal(N), rng.standard_normal(N)
    g[N // 2] = h[N // 2] = 0.0
    g, h = back(dev(g)), back(dev(h))
    t = dev(targets, torch.int32)
    hot = np.zeros((N, M))
    live = (targets >= 0) & (targets < M)
    hot[np.arange(N)[live], targets[live]] = 1
    cp = tylo.allocate_checkpoints_token_logprobs(X)
    fwd = tylo.token_logprobs(X, t, temperature=tau, entropy=True, checkpoints=cp)
    for gg, hh in ((g, h), (g, None), (None, h)):
        z = np.zeros(N)
        ref = oracle.token_logprobs_bwd_ref(z if gg is None else gg, z if hh is None else hh, X64, targets, tau)
        tol = logprob_grad_tolerance(oracle, X64, np.where(live, z if gg is None else gg, 0), z if hh is None else hh, hot, tau, dt, ref)
        tt = None if gg is None else t
        dX = tylo.grad_token_logprobs(None if gg is None else dev(gg), X, tt, checkpoints=cp, temperature=tau,
                                      entropy=fwd.entropy, d_entropy=None if hh is None else dev(hh))
        assert dX.stride(0) == max(X.stride(0), M)
        close(back(dX), ref, tol, "backward")
        out = like(X)
        lp = None if gg is None else tylo.Duplicated(torch.full((N,), 9.0, device="cuda"), dev(gg))
        H = None if hh is None else tylo.Duplicated(torch.full((N,), 9.0, device="cuda"), dev(hh))
        tylo.token_logprobs_with_grad_(lp, tylo.Duplicated(X, out), tt, entropy=H, temperature=tau)
        close(back(out), ref, tol, "one launch")
        if lp is not None:
            close(back(lp.primal), back(fwd.logp), 1e-4, "one launch logp")
        if H is not None:
            close(back(H.primal), back(fwd.entropy), 1e-4, "one launch entropy")
        same = X.clone(memory_format=torch.preserve_format) if pad == 0 else like(X).copy_(X)
        tylo.token_logprobs_with_grad_(lp, tylo.Duplicated(same, same), tt, entropy=H, temperature=tau)
        assert torch.equal(same, out), "in place"
        same.copy_(X)
        grad = None if lp is None else tylo.Duplicated(fwd.logp, lp.shadow)
        tylo.grad_token_logprobs_(grad, tylo.Duplicated(same, same), tt, checkpoints=cp, temperature=tau,
                                  entropy=None if H is None else tylo.Duplicated(fwd.entropy, H.shadow))
        assert torch.equal(same, dX), "backward in place"


def teacher_entries(rng, N, M, K, kind):
    index = np.stack([rng.permutation(M)[:K] if K <= M else rng.integers(0, M, K) for _ in range(N)])
    v = rng.standard_normal((N, K)) * 2 - 1
    if kind == "holes":
        index[rng.random((N, K)) < 0.3] = -1
        index[0] = -1                                # no teacher at all
        index[-1, K // 2] = M
    elif kind == "repeated":
        index[:, K // 2:] = index[:, :1]
    elif kind == "masked":
        v[rng.random((N, K)) < 0.4] = -np.inf
        v[0] = -np.inf
    elif kind == "lowest":                           # entries of the lowest value; a row of nothing else is uniform
        v[rng.random((N, K)) < 0.4] = np.finfo(np.float32).min
        v[0] = np.finfo(np.float32).min
    return v.astype(np.float32).astype(np.float64), index.astype(np.int32)


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("renormalize", [True, False])
@pytest.mark.parametrize("N,M,K,pad,kind,xkind", [
    (1, 1, 1, 0, "plain", "normal"), (7, 9, 9, 0, "plain", "normal"), (5, 1003, 17, 3, "holes", "normal"), (3, 33001, 128, 0, "repeated", "normal"),
    (200, 4096, 64, 8, "masked", "normal"), (4, 20000, 1024, 0, "holes", "lowest"), (6, 300, 1024, 1, "repeated", "masked"),
    (2, 262149, 255, 3, "plain", "large"), (160, 40000, 33, 0, "holes", "normal")])
def test_distillation(tylo, oracle, N, M, K, pad, kind, xkind, renormalize, dt):
    rng = np.random.default_rng(M + K)
    X, X64, _ = logits(rng, N, M, dt, pad=pad, kind=xkind)
    v, index = teacher_entries(rng, N, M, K, kind)
    w = back(dev(rng.standard_normal(N)))
    w[N // 3] = 0.0
    tau, u = 1.7, 1.25
    how = dict(temperature=tau, teacher_temperature=u, renormalize=renormalize)
    V, I, W = dev(v), dev(index, torch.int32), dev(w)
    cp = tylo.allocate_checkpoints_token_logprobs(X)
    loss = tylo.distill(X, V, I, checkpoints=cp, **how)
    logq, q, _, y, rL, _ = row_errors(oracle, X64, tau)
    z, p = oracle._teacher_ref(v, index, M, u, renormalize)
    rp = teacher_tolerance(z, p, K)
    at = np.clip(index, 0, M - 1)
    take = lambda a: np.take_along_axis(a, at, axis=1)
    with np.errstate(invalid="ignore"):
        gap = np.where(p > 0, z - take(logq), 0.0)
        gap = np.where(np.isfinite(gap), np.abs(gap), 0.0)
        zz = np.where(p > 0, np.abs(np.where(np.isfinite(z), z, 0.0)), 0.0)
    tq = logp_tolerance(take(y), rL, take(logq))
    tol = (p * (gap * (rp + (K + 4) * 2.0 ** -24) + tq + rp + zz * 2.0 ** -22)).sum(1)
    ref = oracle.distill_ref(X64, v, index, tau, u, renormalize)
    close(back(loss), ref, tol, "loss")
    dref = oracle.distill_bwd_ref(w, X64, v, index, tau, u, renormalize)
    rq = rL[:, None] + 2.0 ** -22 + 3 * np.abs(y) / np.log(2) * 2.0 ** -24 + 8 * 2.0 ** -24
    P, rP = p.sum(1, keepdims=True), rp.max(1, keepdims=True) + K * 2.0 ** -24
    hot = np.zeros((N, M))
    for n in range(N):
        ok = (index[n] >= 0) & (index[n] < M)
        np.add.at(hot[n], index[n][ok], p[n][ok])
    dtol = (np.abs(w)[:, None] / tau * (q * P * (rq + rP) + hot * (rP + 8 * 2.0 ** -24)) + np.abs(dref) * HALF_STEP[dt] * (1 + 1e-6) + SUBNORMAL[dt])
    dX = tylo.grad_distill(W, X, V, I, checkpoints=cp, **how)
    close(back(dX), dref, dtol, "backward")
    out, l2 = like(X), torch.empty(N, device="cuda")
    tylo.distill_with_grad_(tylo.Duplicated(l2, W), tylo.Duplicated(X, out), V, I, **how)
    close(back(out), dref, dtol, "one launch")
    close(back(l2), ref, tol, "one launch loss")
    same = like(X).copy_(X)
    tylo.distill_with_grad_(tylo.Duplicated(l2, W), tylo.Duplicated(same, same), V, I, **how)
    assert torch.equal(same, out), "in place"
    same.copy_(X)
    tylo.grad_distill_(tylo.Duplicated(loss, W), tylo.Duplicated(same, same), V, I, checkpoints=cp, **how)
    assert torch.equal(same, dX), "backward in place"


@pytest.mark.parametrize("renormalize", [True, False])
def test_teacher_of_the_lowest_value(tylo, oracle, renormalize):
    """A temperature below 1 must not turn the lowest value into -Inf before the largest is taken off."""
    rng = np.random.default_rng(1)
    X, X64, _ = logits(rng, 5, 2000, "f32")
    v, index = teacher_entries(rng, 5, 2000, 40, "lowest")
    how = dict(temperature=1.0, teacher_temperature=0.25, renormalize=renormalize)
    loss, dX = torch.empty(5, device="cuda"), like(X)
    tylo.distill_with_grad_(tylo.Duplicated(loss, dev(np.ones(5))), tylo.Duplicated(X, dX), dev(v), dev(index, torch.int32), **how)
    # 40 terms of order 10 at 2^-20 each; gradients below 1
    np.testing.assert_allclose(back(loss), oracle.distill_ref(X64, v, index, 1.0, 0.25, renormalize), rtol=2.0 ** -18, atol=1e-4)
    np.testing.assert_allclose(back(dX), oracle.distill_bwd_ref(np.ones(5), X64, v, index, 1.0, 0.25, renormalize), rtol=2.0 ** -16, atol=2e-6)


def test_the_longest_row(tylo):
    """One row of 2^31 - 2^16 - 1 logits: indices up to the end of 32 bits.  The reference adds its chunks in 64 bits."""
    M, piece = (1 << 31) - (1 << 16) - 1, 1 << 26
    X = torch.empty(1, M, dtype=torch.float16, device="cuda")
    g = torch.Generator("cuda").manual_seed(2)
    for at in range(0, M, piece):
        n = min(piece, M - at)
        X[0, at:at + n] = torch.randn(n, generator=g, device="cuda", dtype=torch.float16)
    marks = torch.tensor([M - 1, 0, 12345, M // 2 + 1, M - 5, 1 << 30], device="cuda")
    X[0, marks] = torch.tensor([20.0, 19.0, 18.0, 18.0, 17.0, 16.0], dtype=torch.float16, device="cuda")
    total = sum(torch.exp(X[0, at:at + piece].double() - 20.0).sum() for at in range(0, M, piece))
    target = torch.tensor([M - 5], dtype=torch.int32, device="cuda")
    got = tylo.token_logprobs(X, target, top=6)
    assert got.top.index.tolist() == [[M - 1, 0, 12345, M // 2 + 1, M - 5, 1 << 30]]
    # the sum's chains have 2^18 terms (8 CTAs, 512 threads, 2 each): roundings of up to 2^-24 of the sum add up to about 2^9 of them
    # at random, 2^-15; 2^-10 leaves 32 times that
    lse = float(torch.log(total)) + 20.0
    assert abs(float(got.logp) - (17.0 - lse)) < 2.0 ** -10
    w = torch.full((1,), 1024.0, device="cuda")
    lp = torch.empty(1, device="cuda")
    before = X[0, marks].double()
    tylo.token_logprobs_with_grad_(tylo.Duplicated(lp, w), tylo.Duplicated(X, X), target)
    ref = -1024.0 * torch.exp(before - lse)
    ref[4] += 1024.0
    assert torch.allclose(X[0, marks].double(), ref, rtol=2.0 ** -9, atol=2.0 ** -20)


def test_gradients_against_differences(tylo):
    """The kernels' own values, moved by a step in each logit: fp32 differences of a loss of order 1 with step 2^-5 carry
    (2^-20 + chain 2^-24) / 2^-5 of rounding and a curvature of step^2."""
    rng = np.random.default_rng(0)
    M, step = 24, 2.0 ** -5
    x = rng.standard_normal(M)
    rows = np.concatenate([x + step * np.eye(M), x - step * np.eye(M)])
    X, one = dev(rows), dev(x[None])
    t = dev(np.full(2 * M, 5), torch.int32)
    v, index = dev(np.tile(rng.standard_normal(4), (2 * M, 1))), dev(np.tile([3, 5, 5, 20], (2 * M, 1)), torch.int32)
    s = tylo.token_logprobs(X, t, entropy=True)
    for values, grad in (
            (s.logp, lambda cp, f: tylo.grad_token_logprobs(torch.ones(1, device="cuda"), one, t[:1], checkpoints=cp)),
            (s.entropy, lambda cp, f: tylo.grad_token_logprobs(None, one, None, checkpoints=cp, entropy=f.entropy, d_entropy=torch.ones(1, device="cuda"))),
            (tylo.distill(X, v, index), lambda cp, f: tylo.grad_distill(torch.ones(1, device="cuda"), one, v[:1], index[:1], checkpoints=cp))):
        cp = tylo.allocate_checkpoints_token_logprobs(one)
        f = tylo.token_logprobs(one, t[:1], entropy=True, checkpoints=cp)
        values = back(values)
        np.testing.assert_allclose(back(grad(cp, f))[0], (values[:M] - values[M:]) / (2 * step), atol=1e-3)


def test_teacher_to_student(tylo, oracle):
    """The operators as they are used together: a teacher's top alternatives are the entries its student is trained on."""
    rng = np.random.default_rng(3)
    N, M, K, tau = 50, 20001, 32, 1.5
    T, T64, _ = logits(rng, N, M, "bf16")
    S, S64, _ = logits(rng, N, M, "bf16", pad=7)
    top = tylo.token_logprobs(T, temperature=tau, top=K).top
    loss, W = torch.empty(N, device="cuda"), torch.full((N,), 1.0 / N, device="cuda")
    dS = like(S)
    tylo.distill_with_grad_(tylo.Duplicated(loss, W), tylo.Duplicated(S, dS), top.logp, top.index, temperature=tau, teacher_temperature=1.0)
    logp, _, _ = oracle.vocab_stats_ref(T64, tau)
    index = oracle.top_alternatives_ref(T64, K)
    v = np.take_along_axis(logp, index, axis=1)
    np.testing.assert_allclose(back(loss), oracle.distill_ref(S64, v, index, tau, 1.0), rtol=1e-4)
    ref = oracle.distill_bwd_ref(np.full(N, 1.0 / N), S64, v, index, tau, 1.0)
    np.testing.assert_allclose(back(dS), ref, rtol=2.0 ** -7, atol=1e-7)
    # a step against the gradient, then the student's own scores at the teacher's first choice: they rise on average
    before = tylo.token_logprobs(S, top.index[:, 0].contiguous()).logp
    after = tylo.token_logprobs((S.float() - 8.0 * N * dS.float()).to(S.dtype), top.index[:, 0].contiguous()).logp
    assert (after - before).mean() > 0


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("N,M,pad", [(3, 1003, 5), (50, 33001, 1), (2, 200003, 13)])
def test_nothing_outside_the_rows_is_touched(tylo, N, M, pad, dt):
    rng = np.random.default_rng(M)
    X, _, buf = logits(rng, N, M, dt, pad=pad)
    X = X[:N - 1]                                     # a last row that is not part of the call
    before = buf.clone()
    out = torch.full_like(buf, 5.0)
    t, w = torch.zeros(N - 1, dtype=torch.int32, device="cuda"), torch.ones(N - 1, device="cuda")
    v, index = torch.zeros(N - 1, 8, device="cuda"), torch.arange(8, dtype=torch.int32, device="cuda").repeat(N - 1, 1)
    dX = out[:N - 1, :M]
    cp = tylo.allocate_checkpoints_token_logprobs(X)
    tylo.token_logprobs(X, t, top=8, entropy=True, checkpoints=cp)
    tylo.grad_token_logprobs_(tylo.Duplicated(w, w), tylo.Duplicated(X, dX), t, checkpoints=cp)
    tylo.token_logprobs_with_grad_(tylo.Duplicated(w.clone(), w), tylo.Duplicated(X, dX), t)
    tylo.distill_with_grad_(tylo.Duplicated(w.clone(), w), tylo.Duplicated(X, dX), v, index)
    tylo.grad_distill_(tylo.Duplicated(w, w), tylo.Duplicated(X, dX), v, index, checkpoints=cp)
    assert torch.equal(buf, before)
    assert (out[:, M:] == 5.0).all() and (out[N - 1] == 5.0).all()


def test_rows_far_apart(tylo, oracle):
    """Offsets beyond 32 bits of elements: five rows of a buffer of 2.7e9 elements."""
    rng = np.random.default_rng(8)
    ld, M = (1 << 29) + 3, 5001
    buf = torch.empty(5 * ld, dtype=torch.float16, device="cuda")
    X = buf.as_strided((5, M), (ld, 1))
    X.copy_(dev(rng.standard_normal((5, M)) * 3, torch.float16))
    targets = rng.integers(0, M, 5)
    got, cp = check_score(tylo, oracle, X, back(X), targets, 1.0, 16, "far rows")
    del got
    X64 = back(X)
    w = dev(np.ones(5))
    tylo.grad_token_logprobs_(tylo.Duplicated(w, w), tylo.Duplicated(X, X), dev(targets, torch.int32), checkpoints=cp)
    ref = oracle.token_logprobs_bwd_ref(np.ones(5), np.zeros(5), X64, targets)
    np.testing.assert_allclose(back(X), ref, atol=2.0 ** -11)


def test_captured_replayed_and_on_another_stream(tylo):
    rng = np.random.default_rng(4)
    N, M, K = 20, 50001, 64
    X, _, _ = logits(rng, N, M, "bf16", pad=7)
    t, w = dev(rng.integers(0, M, N), torch.int32), dev(rng.standard_normal(N))

    def buffers():
        return dict(lp=torch.empty(N, device="cuda"), H=torch.empty(N, device="cuda"), top=tylo.allocate_top_alternatives(X, K), dX=like(X),
                    loss=torch.empty(N, device="cuda"), dS=like(X), cp=tylo.allocate_checkpoints_token_logprobs(X))

    def step(b):
        tylo.token_logprobs_(b["lp"], X, t, entropy=b["H"], top=b["top"], checkpoints=b["cp"])
        tylo.grad_token_logprobs_(tylo.Duplicated(b["lp"], w), tylo.Duplicated(X, b["dX"]), t, checkpoints=b["cp"], entropy=tylo.Duplicated(b["H"], w))
        tylo.distill_with_grad_(tylo.Duplicated(b["loss"], w), tylo.Duplicated(X, b["dS"]), b["top"].logp, b["top"].index)

    want = buffers()
    step(want)
    torch.cuda.synchronize()
    got = [buffers(), buffers()]
    streams, graphs = [torch.cuda.Stream(), torch.cuda.Stream()], [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()]
    for b, s, g in zip(got, streams, graphs):
        with torch.cuda.graph(g, stream=s):
            step(b)
    X.mul_(0.5)                                       # a replay reads what is there when it runs
    step(want)
    torch.cuda.synchronize()
    for s, g in zip(streams, graphs):                 # both in flight at once
        with torch.cuda.stream(s):
            g.replay()
            g.replay()
    torch.cuda.synchronize()
    for b in got:
        for k in want:
            for x, y in zip(want[k] if isinstance(want[k], tuple) else [want[k]], b[k] if isinstance(b[k], tuple) else [b[k]]):
                assert torch.equal(x, y), k


def test_calls_of_several_threads(tylo):
    """Rows of different lengths that take the same kernel, whose needs of shared memory differ, from threads that run at once."""
    lengths = (34000, 40000, 47000, 54000)
    rng = np.random.default_rng(12)
    data = []
    for M in lengths:
        X, _, _ = logits(rng, 600, M, "bf16")
        t, g = dev(rng.integers(0, M, 600), torch.int32), torch.ones(600, device="cuda")
        teacher, index = dev(rng.standard_normal((600, 4))), dev(rng.integers(0, M, (600, 4)), torch.int32)
        data.append((X, t, g, teacher, index))

    def both(X, t, g, teacher, index):
        logp, loss, d1, d2 = torch.empty_like(g), torch.empty_like(g), torch.empty_like(X), torch.empty_like(X)
        tylo.token_logprobs_with_grad_(tylo.Duplicated(logp, g), tylo.Duplicated(X, d1), t)
        tylo.distill_with_grad_(tylo.Duplicated(loss, g), tylo.Duplicated(X, d2), teacher, index)
        return logp, loss, d1, d2

    want = [both(*d) for d in data]
    torch.cuda.synchronize()
    start = threading.Barrier(len(data))

    def work(i):
        start.wait(60)
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(100):
                got = both(*data[i])
            torch.cuda.current_stream().synchronize()
            return all(torch.equal(a, b) for a, b in zip(got, want[i]))

    with ThreadPoolExecutor(len(data)) as pool:
        assert all(pool.map(work, range(len(data))))


@pytest.mark.parametrize("N,M", [(1, 131072), (33, 50001), (400, 8192)])
def test_equal_inputs_give_equal_bits(tylo, N, M):
    rng = np.random.default_rng(N)
    X, _, _ = logits(rng, N, M, "bf16", kind="ties")
    t, w = dev(rng.integers(0, M, N), torch.int32), dev(rng.standard_normal(N))
    index = dev(rng.integers(0, M, (N, 64)), torch.int32)
    index[:, 32:] = index[:, :32]
    v = dev(rng.standard_normal((N, 64)))
    runs = []
    for _ in range(3):
        a = tylo.token_logprobs(X, t, entropy=True, top=128)
        dX, dS, loss = torch.empty_like(X), torch.empty_like(X), torch.empty(N, device="cuda")
        tylo.token_logprobs_with_grad_(tylo.Duplicated(loss.clone(), w), tylo.Duplicated(X, dX), t)
        tylo.distill_with_grad_(tylo.Duplicated(loss, w), tylo.Duplicated(X, dS), v, index)
        runs.append([a.logp, a.entropy, a.top.logp, a.top.index, dX, dS, loss])
    for r in runs[1:]:
        assert all(torch.equal(x, y) for x, y in zip(runs[0], r))


def test_refusals(tylo):
    X = torch.zeros(4, 64, device="cuda")
    t, f = torch.zeros(4, dtype=torch.int32, device="cuda"), torch.zeros(4, device="cuda")
    bad = [lambda: tylo.token_logprobs(X.cpu(), t), lambda: tylo.token_logprobs(X, t.long()), lambda: tylo.token_logprobs(X, t[:3].contiguous()),
           lambda: tylo.token_logprobs(X.t(), t), lambda: tylo.token_logprobs(X[0], t), lambda: tylo.token_logprobs(X, t.cpu()),
           lambda: tylo.token_logprobs_(f.double(), X, t), lambda: tylo.distill(X, torch.zeros(4, 2, device="cuda"), t),
           lambda: tylo.distill(X, torch.zeros(4, 2, device="cuda").half(), torch.zeros(4, 2, dtype=torch.int32, device="cuda")),
           lambda: tylo.grad_token_logprobs_(tylo.Duplicated(f, f), tylo.Duplicated(X, torch.zeros(4, 80, device="cuda")[:, :64]), t,
                                             checkpoints=tylo.allocate_checkpoints_token_logprobs(X)),
           lambda: tylo.grad_token_logprobs_(tylo.Duplicated(f, f), tylo.Duplicated(X, X.half()), t, checkpoints=tylo.allocate_checkpoints_token_logprobs(X)),
           lambda: tylo.token_logprobs(X[:, :64].expand(4, 64)[:1].expand(4, 64), t)]
    for call in bad:
        with pytest.raises(ValueError):
            call()
    with pytest.raises(TypeError):
        tylo.token_logprobs(X.double(), t)
    for call, status in ((lambda: tylo.token_logprobs(X, t, top=65), 1), (lambda: tylo.token_logprobs(torch.zeros(4, 512, device="cuda"), t, top=257), 1),
                         (lambda: tylo.token_logprobs(X, t, temperature=0.0), 1), (lambda: tylo.token_logprobs(X, t, temperature=float("nan")), 1),
                         (lambda: tylo.token_logprobs(X), 1), (lambda: tylo.token_logprobs(X.view(-1)[1:193].view(3, 64), t[:3].contiguous()), 3)):
        with pytest.raises(tylo.TyloError) as e:
            call()
        assert e.value.status == status
