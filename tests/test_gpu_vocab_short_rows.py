"""GPU: top alternatives of rows of which fewer threads hold data than there are alternatives, but more elements than the selection has
places for: the bound that the threads' maxima give is then below every element.  16-byte packets, so 16-bit types reach this from 513
logits with 128 threads (many rows, up to 64 alternatives), from 1025 with 256 threads and from 2049 with 512.  Rows an odd number of
elements apart begin at every place of a packet.  The indices have to be the oracle's, the log probabilities within the tolerance that
vocab_util.py derives."""
import numpy as np
import pytest
import torch

from test_gpu_vocab import check_score, logits

pytestmark = pytest.mark.gpu


def run(tylo, oracle, N, M, tops, dt, kind):
    rng = np.random.default_rng(M + N)
    X, X64, _ = logits(rng, N, M, dt, kind=kind, pad=1 + M % 2)         # an odd distance between the rows
    assert X.stride(0) % 2 == 1
    targets = rng.integers(-1, M, N)
    for K in tops:
        got, _ = check_score(tylo, oracle, X, X64, targets, 1.0, K, f"{M} logits, {K} alternatives")
        again = tylo.token_logprobs(X, top=K).top
        assert torch.equal(again.index, got.top.index)


@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("kind", ["normal", "masked", "lowest", "ties"])
@pytest.mark.parametrize("M", [1023, 1025, 1026, 1030, 1100, 1300, 1408, 1415, 1423])
def test_256_threads(tylo, oracle, M, kind, dt):
    run(tylo, oracle, 9, M, (64, 65, 127, 128, 129, 137, 150, 163, 176, 177), dt, kind)


@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("kind", ["normal", "masked", "lowest", "ties"])
@pytest.mark.parametrize("M", [1500, 2047, 2049, 2050, 2054, 2060, 2100])
def test_512_threads(tylo, oracle, M, kind, dt):
    run(tylo, oracle, 9, M, (176, 177, 200, 255, 256), dt, kind)


@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("kind", ["normal", "masked", "ties"])
@pytest.mark.parametrize("M", [511, 513, 514, 516, 518, 520])
def test_128_threads(tylo, oracle, M, kind, dt):
    run(tylo, oracle, 1500, M, (63, 64, 65), dt, kind)


@pytest.mark.parametrize("dt", ["bf16", "f16"])
@pytest.mark.parametrize("M,K", [(1100, 150), (1026, 128), (2051, 256)])
def test_with_nan_and_infinities(tylo, oracle, M, K, dt):
    rng = np.random.default_rng(M)
    X, _, _ = logits(rng, 9, M, dt, pad=1 + M % 2)
    X[0, M // 2] = float("nan")
    X[1, [0, M - 1]] = float("nan")
    X[2, 5] = float("inf")
    X[3] = float("-inf")
    X[4] = float("-inf")
    X[4, 7] = float("nan")
    X[5, 3:] = float("-inf")
    X[6, 1::2] = float("-inf")
    X[7] = float("nan")
    index = tylo.token_logprobs(X, top=K).top.index
    assert np.array_equal(index.cpu().numpy(), oracle.top_alternatives_ref(X.double().cpu().numpy(), K))
