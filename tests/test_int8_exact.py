"""What the exact data of int8_exact.py can tell apart, on the CPU: mistakes planted in the oracle have to change
its result at every size that the GPU tests run."""
import pytest
import torch

import int8_exact as X
from test_gpu_int8_exact import EXACT, TYPES


def _in_parts(a, parts):
    """Scaled gradients as `parts` fp16 parts, as the kernels take them."""
    power = torch.exp2(14 - torch.floor(torch.log2(torch.stack([v.abs().amax(1) for v in a]).amax(0))))[:, None]
    out = []
    for v in a:
        left, kept = v * power, torch.zeros_like(v)
        for t in range(parts):
            h = left.half().double()
            kept, left = kept + h * 2.0 ** (-11 * t), (left - h) * 2048
        out.append(kept / power)
    return out


def _without(a, lo, hi, bank=-1):
    b = [v.clone() for v in a]
    b[bank][:, lo:hi] = 0
    return b


def _cases(M, K, N, t, dense):
    m, k = min(M, 12), min(K, 160)
    dy, w, s = X.product_case(m, N, k, t, dense, "cpu")
    yield X.scaled([dy], [s]), [w]
    dy, gate, up, w, s = X.gated_case(m, N, k, t, dense, "cpu")
    yield X.scaled([dy.double() * up.double(), dy.double() * gate.double()], s), w


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("M,K,N", EXACT)
def test_a_lost_term_shows(M, K, N, t):
    for a, w in _cases(M, K, N, t, True):
        right = X.rounded(X.exact_sum(a, w), t)
        step = (N - 1) // 64 * 64  # the last, ragged step of 64
        for bank in range(len(a)):
            for lo, hi in ((N - 1, N), (step, N), (0, 1), (0, 64), (step // 128 * 64, step // 128 * 64 + 64)):
                assert not torch.equal(X.rounded(X.exact_sum(_without(a, lo, hi, bank), w), t), right), (bank, lo, hi)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("M,K,N", EXACT)
def test_a_lost_part_shows(M, K, N, t):
    parts = 3 if t == torch.float32 else 2
    for a, w in _cases(M, K, N, t, False):
        right = X.exact_sum(a, w)
        as_parts = lambda n: sum(v @ c.double() for v, c in zip(_in_parts(a, n), w)).float().to(t)
        assert torch.equal(as_parts(parts), X.rounded(right, t))
        if t != torch.bfloat16:  # (its own 8 bits hide most of what one part loses: what is left is in the next test)
            assert not torch.equal(as_parts(parts - 1), X.rounded(right, t))
        assert not torch.equal(X.rounded(X.exact_sum(_without(a, N - 2, N), w), t), X.rounded(right, t))


@pytest.mark.parametrize("t", TYPES)
def test_a_lost_part_is_over_the_bounds(t):
    dy, w, s = X.cancelling_case(130, 400, t, "cpu")
    ref, tol = X.cancelling_sum(dy, w, s, 2.0 ** -22)
    a = X.scaled([dy], [s])
    off = lambda n: ((_in_parts(a, n)[0] @ w.double()).float().to(t).double() - ref).abs() - tol
    assert off(2).max() <= 0 < off(1).max()
    dy, w, s = X.wide_case(130, 400, 28, "cpu")
    ref = dy.double() @ w.double()
    err = lambda n: ((_in_parts([dy.double()], n)[0] @ w.double()) / ref - 1).abs().max().item()
    assert err(3) == 0.0 < err(2) <= 2.0 ** -22 < err(1)
