"""CPU: the vocabulary entry points check their arguments before touching a device (nothing is launched)."""
import ctypes

import pytest


def f(n=1):
    return ctypes.c_void_p(0x1000 * n)       # aligned, never dereferenced: the check fails first


def _fwd(lib, Logp=f(1), Entropy=None, TopLogp=None, TopIndex=None, Mx=None, L=None, X=f(2), targets=f(3), top=0, M=64, N=4, ld=64, tau=1.0, dtype=0):
    return lib.tylo_b200_token_logprobs_fwd(Logp, Entropy, TopLogp, TopIndex, Mx, L, X, targets, top, M, N, ld, tau, dtype, None)


@pytest.mark.parametrize("change,status,word", [
    (dict(X=None), 1, b"X"), (dict(M=0), 1, b"positive"), (dict(N=0), 1, b"positive"), (dict(ld=63), 1, b"ldx"), (dict(tau=0.0), 1, b"temperature"),
    (dict(tau=-1.0), 1, b"temperature"), (dict(tau=float("nan")), 1, b"temperature"), (dict(tau=float("inf")), 1, b"temperature"),
    (dict(X=ctypes.c_void_p(0x1008)), 3, b"16-byte"), (dict(targets=None), 1, b"targets"), (dict(Logp=None), 1, b"nothing"),
    (dict(Logp=None, Entropy=f(5)), 1, b"targets"), (dict(Mx=f(4)), 1, b"together"), (dict(top=1), 1, b"TopLogp"), (dict(TopLogp=f(4), TopIndex=f(5)), 1, b"top"),
    (dict(top=-1), 1, b"top"), (dict(top=65, TopLogp=f(4), TopIndex=f(5)), 1, b"at most M"),
    (dict(top=257, M=512, ld=512, TopLogp=f(4), TopIndex=f(5)), 1, b"256"), (dict(dtype=3), 1, b"dtype"), (dict(dtype=9), 1, b"dtype"),
    (dict(M=1 << 31, ld=1 << 31), 2, b"not supported"), (dict(N=1 << 30), 2, b"not supported"), (dict(ld=(1 << 34) + 1), 2, b"not supported")])
def test_scores(tylo, change, status, word):
    assert _fwd(tylo._lib, **change) == status
    assert word in tylo._lib.tylo_b200_last_error()


def test_score_gradients(tylo):
    lib = tylo._lib
    err = lib.tylo_b200_last_error
    bwd = lambda dX=f(1), g=f(2), h=None, X=f(3), t=f(4), H=None, m=f(5), L=f(6), M=64, N=4, ld=64, tau=1.0: \
        lib.tylo_b200_token_logprobs_bwd(dX, g, h, X, t, H, m, L, M, N, ld, tau, 0, None)
    assert bwd(dX=None) == 1 and b"dX" in err()
    assert bwd(dX=ctypes.c_void_p(0x1004)) == 3
    assert bwd(t=None) == 1 and b"targets" in err()
    assert bwd(g=None, t=None) == 1 and b"dEntropy" in err()
    assert bwd(h=f(7)) == 1 and b"Entropy" in err()
    assert bwd(m=None) == 1 and b"checkpoints" in err()
    assert bwd(ld=10) == 1 and b"ldx" in err()
    both = lambda lp=f(1), H=None, dX=f(2), g=f(3), h=None, X=f(4), t=f(5): \
        lib.tylo_b200_token_logprobs_fwd_bwd(lp, H, dX, g, h, X, t, 64, 4, 64, 1.0, 0, None)
    assert both(dX=None) == 1
    assert both(g=None) == 1 and b"targets" in err()
    assert both(g=None, t=None, h=f(6)) == 1 and b"Logp" in err()
    assert both(g=None, t=None) == 1


def test_distillation(tylo):
    lib = tylo._lib
    err = lib.tylo_b200_last_error
    fwd = lambda loss=f(1), m=None, L=None, X=f(2), v=f(3), i=f(4), K=8, M=64, N=4, ld=64, tau=1.0, u=1.0, dt=0: \
        lib.tylo_b200_distill_fwd(loss, m, L, X, v, i, K, M, N, ld, tau, u, 1, dt, None)
    assert fwd(loss=None) == 1 and b"Loss" in err()
    assert fwd(v=None) == 1 and b"teacher" in err()
    assert fwd(i=None) == 1
    assert fwd(K=0) == 1 and fwd(K=1025) == 1 and b"1024" in err()
    assert fwd(u=0.0) == 1 and b"teacher_temperature" in err()
    assert fwd(L=f(5)) == 1 and b"together" in err()
    assert fwd(dt=7) == 1
    assert lib.tylo_b200_distill_bwd(f(1), None, f(2), f(3), f(4), f(5), f(6), 8, 64, 4, 64, 1.0, 1.0, 1, 0, None) == 1
    assert lib.tylo_b200_distill_bwd(f(1), f(7), f(2), f(3), f(4), None, f(6), 8, 64, 4, 64, 1.0, 1.0, 1, 0, None) == 1 and b"checkpoints" in err()
    assert lib.tylo_b200_distill_fwd_bwd(f(1), None, f(7), f(2), f(3), f(4), 8, 64, 4, 64, 1.0, 1.0, 1, 0, None) == 1
    assert lib.tylo_b200_distill_fwd_bwd(f(1), ctypes.c_void_p(0x1008), f(7), f(2), f(3), f(4), 8, 64, 4, 64, 1.0, 1.0, 1, 0, None) == 3


def test_overlapping_arrays_are_refused(tylo):
    lib = tylo._lib
    err = lib.tylo_b200_last_error
    at = ctypes.c_void_p
    # 4 rows of 64 fp32 logits, 256 elements apart: the gradient shifted by 16 bytes, by a row, into the gap (the check behind it fails)
    bwd = lambda dX, M=64, ld=256, N=4, dt=0: lib.tylo_b200_token_logprobs_bwd(at(dX), f(2), None, at(0x100000), f(4), None, None, None, M, N, ld, 1.0, dt, None)
    for dX in (0x100010, 0x100000 - 16, 0x100000 + 4 * 256, 0x100000 - 4 * 256, 0x100000 + 4 * 60, 0x100000 + 4 * (3 * 256 + 60)):
        assert bwd(dX) == 1 and b"overlap" in err()
    for dX in (0x100000, 0x100000 + 4 * 64, 0x100000 + 4 * 192, 0x100000 + 4 * (3 * 256 + 64), 0x100000 - 4 * (3 * 256 + 64)):
        assert bwd(dX) == 1 and b"checkpoints" in err()
    assert bwd(0x100000 + 2 * 64, dt=1) == 1 and b"checkpoints" in err()
    assert bwd(0x100000 + 2 * 56, dt=1) == 1 and b"overlap" in err()
    w = f(9)
    assert lib.tylo_b200_token_logprobs_fwd_bwd(w, None, f(2), w, None, f(3), f(4), 64, 4, 64, 1.0, 0, None) == 1 and b"different" in err()
    assert lib.tylo_b200_distill_fwd_bwd(w, f(2), w, f(3), f(4), f(5), 8, 64, 4, 64, 1.0, 1.0, 1, 0, None) == 1 and b"different" in err()
    assert lib.tylo_b200_distill_bwd(at(0x3010), w, f(3), f(4), f(5), f(6), f(7), 8, 64, 4, 64, 1.0, 1.0, 1, 0, None) == 1 and b"overlap" in err()


def test_host_arrays_are_refused(tylo):
    import torch
    X, t, w = torch.zeros(4, 64), torch.zeros(4, dtype=torch.int32), torch.zeros(4)
    v, i = torch.zeros(4, 2), torch.zeros(4, 2, dtype=torch.int32)
    cp = tylo.allocate_checkpoints_token_logprobs(X)
    dup = tylo.Duplicated
    for call in (lambda: tylo.token_logprobs(X, t, entropy=True, top=3), lambda: tylo.grad_token_logprobs(w, X, t, checkpoints=cp),
                 lambda: tylo.token_logprobs_with_grad_(dup(w, w), dup(X, X), t), lambda: tylo.distill(X, v, i),
                 lambda: tylo.grad_distill(w, X, v, i, checkpoints=cp), lambda: tylo.distill_with_grad_(dup(w, w), dup(X, X), v, i)):
        with pytest.raises(ValueError, match="device"):
            call()
