"""CPU: the oracle of the vocabulary scores and losses against torch autograd in float64, against differences, and on rows that a mask
leaves empty."""
import numpy as np
import pytest
import torch


def _inputs(N=5, M=23, K=4, seed=0):
    rng = np.random.default_rng(seed)
    X = rng.standard_normal((N, M)) * 2
    t = rng.integers(0, M, N)
    index = np.stack([rng.permutation(M)[:K] for _ in range(N)])
    return rng, X, t, rng.standard_normal((N, K)), index


@pytest.mark.parametrize("tau", [1.0, 0.6, 2.0])
def test_logprobs_and_gradient_match_autograd(oracle, tau):
    rng, X, t, _, _ = _inputs()
    g, h = rng.standard_normal(5), rng.standard_normal(5)
    x = torch.tensor(X, requires_grad=True)
    lp = torch.log_softmax(x / tau, 1)
    logp, H = lp[torch.arange(5), torch.tensor(t)], -(lp.exp() * lp).sum(1)
    (logp @ torch.tensor(g) + H @ torch.tensor(h)).backward()
    rl, rH = oracle.token_logprobs_ref(X, t, tau)
    np.testing.assert_allclose(rl, logp.detach().numpy(), rtol=1e-12)
    np.testing.assert_allclose(rH, H.detach().numpy(), rtol=1e-12)
    np.testing.assert_allclose(oracle.token_logprobs_bwd_ref(g, h, X, t, tau), x.grad.numpy(), rtol=1e-10, atol=1e-13)


@pytest.mark.parametrize("renormalize", [True, False])
def test_distill_and_gradient_match_autograd(oracle, renormalize):
    rng, X, _, v, index = _inputs()
    index[0, 1] = -1
    index[1, 2] = 23
    index[2, 3] = index[2, 0]                      # the same token twice
    w, tau, u = rng.standard_normal(5), 1.7, 0.8
    x = torch.tensor(X, requires_grad=True)
    live = torch.tensor((index >= 0) & (index < 23))
    z = torch.where(live, torch.tensor(v) / u, -torch.inf)
    z = torch.log_softmax(z, 1) if renormalize else z
    logq = torch.log_softmax(x / tau, 1).gather(1, torch.tensor(np.clip(index, 0, 22)))
    loss = torch.where(live, z.exp() * (torch.where(live, z, 0.0) - logq), 0.0).sum(1)
    (loss @ torch.tensor(w)).backward()
    np.testing.assert_allclose(oracle.distill_ref(X, v, index, tau, u, renormalize), loss.detach().numpy(), rtol=1e-12)
    np.testing.assert_allclose(oracle.distill_bwd_ref(w, X, v, index, tau, u, renormalize), x.grad.numpy(), rtol=1e-10, atol=1e-13)


def test_gradients_match_differences(oracle):
    rng, X, t, v, index = _inputs(N=2, M=7, K=3)
    g, h, e = rng.standard_normal(2), rng.standard_normal(2), 1e-6
    f = lambda X: oracle.token_logprobs_ref(X, t, 0.7)[0] @ g + oracle.token_logprobs_ref(X, t, 0.7)[1] @ h
    d = lambda X: oracle.distill_ref(X, v, index, 0.7) @ g
    for fn, grad in ((f, oracle.token_logprobs_bwd_ref(g, h, X, t, 0.7)), (d, oracle.distill_bwd_ref(g, X, v, index, 0.7))):
        for i in np.ndindex(X.shape):
            hi, lo = X.copy(), X.copy()
            hi[i] += e
            lo[i] -= e
            assert abs((fn(hi) - fn(lo)) / (2 * e) - grad[i]) < 1e-7


def test_empty_rows_padding_and_ties(oracle):
    X = np.array([[-np.inf] * 4, [1.0, 3.0, 3.0, -np.inf], [-np.inf, 0.0, -np.inf, -np.inf], [np.nan, 1.0, 2.0, np.nan]])
    logp, H = oracle.token_logprobs_ref(X[:3], [2, -1, 1])
    assert np.isneginf(logp[0]) and logp[1] == 0 and logp[2] == 0 and H[0] == 0 and H[2] == 0
    assert oracle.top_alternatives_ref(X, 3).tolist() == [[0, 1, 2], [1, 2, 0], [1, 0, 2], [0, 3, 2]]
    d = oracle.token_logprobs_bwd_ref([1.0, 1.0, 1.0], [1.0, 0.0, 1.0], X[:3], [2, 4, 1])
    assert (d[0] == 0).all() and (d[1] == 0).all() and (d[2] == 0).all()
    v, index = np.zeros((3, 2)), np.array([[0, 1], [-1, 9], [1, 1]])
    loss = oracle.distill_ref(X[:3], v, index)
    assert np.isposinf(loss[0]) and loss[1] == 0 and loss[2] == pytest.approx(-np.log(2))
    d = oracle.distill_bwd_ref(np.ones(3), X[:3], v, index)
    assert (d == 0).all()
