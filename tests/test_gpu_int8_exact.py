"""The int8 operators on data with one right answer (int8_exact.py), and in the kernels that the other sizes miss."""
import math

import pytest
import torch

import int8_exact as X
import int8_ref as R
import mi_qmm

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
TYPES = [BF16, F16, F32]


def _case(**kw):
    print("CASE", kw, flush=True)


def _off(t, n):
    """The same values n elements behind a 16-byte boundary."""
    v = torch.empty(t.numel() + n, dtype=t.dtype, device="cuda")[n:].view(t.shape)
    v.copy_(t)
    return v


def _within(y, ref, tol, what):
    over = (y.double() - ref).abs() - tol
    assert torch.isfinite(y).all() and over.max().item() <= 0, f"{what}: {over.max().item():.3g} over the bound"


# ------------------------------------------------ what a scaled gradient keeps --
@pytest.mark.parametrize("M,N", [(1, 16), (5, 48), (130, 208), (300, 1000)])
def test_fp32_gradients_keep_22_bits(dev, M, N):
    """Down to 2^-28 of their row's largest value."""
    _case(t="wide", M=M, N=N)
    dy, w, s = X.wide_case(M, N, 28, "cuda")
    ref = dy.double() @ w.double()
    for what, args in (("aligned", (dy, w, s)), ("off", (_off(dy, 1), _off(w, 3), s))):
        _within(mi_qmm.int8_matmul_backward(*args), ref, 2.0 ** -22 * ref.abs(), what)


@pytest.mark.parametrize("M,N", [(1, 16), (5, 48), (130, 208), (300, 1000)])
def test_fp32_gradients_keep_all_bits(dev, M, N):
    """24 bits of each value down to 2^-28 of their row's largest, in a row that goes down to 2^-37.

    Below 2^-28 the first part is subnormal. The matrix instruction adds what the smaller parts gave to a product
    that it places by the smallest normal exponent, less than 2 x 2^-14 |w|; of what is added 24 bits from there
    stay, which cuts off less than 2^-37 |w|. The row's largest is 2^14 at least: 2^-51 |w| of it. The second part
    does the same 2^-11 lower, and 2^-61 was not kept at all: 2^-50 in all."""
    _case(t="all bits", M=M, N=N)
    dy, w, s = X.wide_case(M, N, 37, "cuda")
    ref = dy.double() @ w.double()
    top = dy.abs().amax(1, keepdim=True)
    small = dy.abs() < top * 2.0 ** -28  # (w is a diagonal: column k has dy[:, k])
    tol = torch.where(small, 2.0 ** -50 * top.double() * w.double().abs().sum(0), 0.0)
    assert small.sum() < 0.4 * small.numel()
    for what, args in (("aligned", (dy, w, s)), ("off", (_off(dy, 1), _off(w, 3), s))):
        _within(mi_qmm.int8_matmul_backward(*args), ref, tol, what)


@pytest.mark.parametrize("M,N", [(5, 48), (130, 208)])
def test_banks_of_unlike_scales(dev, M, N):
    """dup's scales 2^-24 of dgate's: its part of dx keeps 22 bits, though both share a row's power of two."""
    dy, w, s = X.wide_case(M, N, 3, "cuda")
    z = torch.zeros_like(w)
    gate, up = torch.full_like(dy, 64.0), torch.ones_like(dy)
    wg, wu = torch.cat([w, z], 1), torch.cat([z, w], 1)
    su = s * 2.0 ** -30
    dx, dg, du = mi_qmm.int8_gate_up_swiglu_backward(dy, gate, up, wg, s, wu, su)
    assert torch.equal(dg, dy) and torch.equal(du, 64 * dy)
    ref = torch.cat([dy.double() @ w.double(), (64 * dy.double() * su.double()) @ w.double()], 1)
    _within(dx, ref, 2.0 ** -22 * ref.abs(), "dx")


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("M,N", [(3, 32), (130, 400), (300, 2080)])
def test_differences_of_products(dev, M, N, t):
    """Two products a column that nearly cancel: 22 bits of each."""
    _case(t="differences", M=M, N=N, type=t)
    dy, w, s = X.cancelling_case(M, N, t, "cuda")
    ref, tol = X.cancelling_sum(dy, w, s, 2.0 ** -22)
    for what, args in (("aligned", (dy, w, s)), ("off", (_off(dy, 1), _off(w, 3), s))):
        _within(mi_qmm.int8_matmul_backward(*args), ref, tol, what)
    gate, up, z = torch.full_like(dy, 64.0), torch.ones_like(dy), torch.zeros_like(w)
    _within(mi_qmm.int8_gate_up_swiglu_backward(dy, gate, up, w, s, z, s / 64)[0], ref, tol, "gate + up")


# ------------------------------------------------------ sums with one right answer --
# Every tile of the product, with and without ranges of the sum, and the small tiles behind whole rounds of big ones, for
# each count of banks and parts; rows, columns and the sum end inside tiles and steps.
EXACT = [(18, 36, 65), (1477, 119, 65), (2103, 34, 337), (2716, 652, 72), (2719, 656, 130), (66, 8650, 838),
         (70, 8656, 900), (2091, 1940, 193), (2091, 1944, 200), (129, 3278, 5450), (129, 3280, 5452), (150, 6551, 6739),
         (2712, 8553, 194), (2712, 8560, 200), (667, 4100, 4096), (1000, 2048, 5632), (512, 14336, 4096),
         (1024, 4096, 14336)]


@pytest.mark.parametrize("dense", [True, False])
@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("M,K,N", EXACT)
def test_exact_product_gradients(dev, M, K, N, t, dense):
    _case(t="exact", M=M, K=K, N=N, type=t, dense=dense)
    dy, w, s = X.product_case(M, N, K, t, dense, "cuda")
    want = X.rounded(X.exact_sum(X.scaled([dy], [s]), [w]), t)
    assert torch.equal(mi_qmm.int8_matmul_backward(dy, w, s), want)


@pytest.mark.parametrize("dense", [True, False])
@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("M,K,N", EXACT)
def test_exact_gated_gradients(dev, M, K, N, t, dense):
    _case(t="exact gated", M=M, K=K, N=N, type=t, dense=dense)
    dy, gate, up, w, s = X.gated_case(M, N, K, t, dense, "cuda")
    d = [dy.double() * up.double(), dy.double() * 64]
    want = X.rounded(X.exact_sum(X.scaled(d, s), w), t)
    dx, dg, du = mi_qmm.int8_gate_up_swiglu_backward(dy, gate, up, w[0], s[0], w[1], s[1])
    assert torch.equal(dx, want)
    assert torch.equal(dg, X.rounded(d[0], t)) and torch.equal(du, X.rounded(d[1], t))


# ------------------------------------------------------------------- the sigmoid --
def test_silu_in_fp32(dev):
    x, sx, wg, sg, wu, su = X.silu_case("cuda")
    ref, tol = X.silu(x, wg, sg, wu, su)
    for m in (1, 40, x.shape[0]):
        y = mi_qmm.int8_gate_up_swiglu(x[:m].contiguous(), wg, sg, wu, su, x_scales=sx[:m].contiguous(), dtype=F32)
        _within(y, ref[:m], tol[:m], m)


def test_silu_gradient_in_fp32(dev):
    g = torch.cat([torch.arange(-6400, 6400, device="cuda").float() / 64, torch.tensor([-1.2784645, 0.0], device="cuda")])
    gate = torch.cat([g, g[:14]]).view(-1, 16)  # 801 rows
    r = X.gen(1, "cuda")
    dy, up = (torch.randn(gate.shape, device="cuda", generator=r) for _ in range(2))
    w, s = torch.ones(16, 32, dtype=torch.int8, device="cuda"), torch.ones(16, device="cuda")
    ref_g, ref_u, tol_g, tol_u = X.dsilu(dy, gate, up)
    for args in ((dy, gate, up), (_off(dy, 1), gate, up)):
        _, dg, du = mi_qmm.int8_gate_up_swiglu_backward(*args, w, s, w, s)
        _within(dg, ref_g, tol_g, "dgate")
        _within(du, ref_u, tol_u, "dup")


# ---------------------------------------------- kernels that other sizes miss --
def _codes(M, N, K, banks):
    g = X.gen(M + N + K, "cuda")
    ints = lambda n: torch.randint(-127, 128, (n, K), device="cuda", generator=g, dtype=torch.int32).to(torch.int8)
    return (ints(M), torch.rand(M, device="cuda", generator=g) + 0.1, [ints(N) for _ in range(banks)],
            [torch.rand(N, device="cuda", generator=g) * 1e-3 + 1e-5 for _ in range(banks)],
            torch.randn(N, device="cuda", generator=g))


@pytest.mark.parametrize("t,K", [(BF16, 4112), (BF16, 14336), (BF16, 16384), (F16, 5632), (F16, 14336), (F32, 2064),
                                 (F32, 8192)])
def test_long_float_token(dev, t, K):
    """One token of more than 8 KB, quantized in the launch: four vectors a thread."""
    _case(t="token", K=K, type=t)
    g = X.gen(K, "cuda")
    x = torch.randn(1, K, device="cuda", generator=g).to(t)
    x[0, K - 1] = 9.0  # the row's largest value sits at its end
    w = [torch.randint(-127, 128, (100, K), device="cuda", generator=g, dtype=torch.int32).to(torch.int8) for _ in range(2)]
    s = [torch.rand(100, device="cuda", generator=g) * 1e-3 + 1e-5 for _ in range(2)]
    q, sx = R.quantize(x)
    ref, tol = R.matmul(q, sx, w[0], s[0])
    y = mi_qmm.int8_matmul(x, w[0], s[0])
    R.check(y, ref, tol(t), "y")
    assert torch.equal(y, mi_qmm.int8_matmul(q, w[0], s[0], x_scales=sx, dtype=t))
    assert torch.equal(y, mi_qmm.int8_matmul(_off(x, 1), w[0], s[0]))
    h = mi_qmm.int8_gate_up_swiglu(x, w[0], s[0], w[1], s[1], save=True)
    r = R.gate_up(q, sx, w[0], s[0], w[1], s[1])
    for a, b, e in zip(h, r[:3], r[3:]):
        R.check(a, b, e(t), "gate + up")
    h2 = mi_qmm.int8_gate_up_swiglu(q, w[0], s[0], w[1], s[1], x_scales=sx, dtype=t, save=True)
    assert all(torch.equal(a, b) for a, b in zip(h, h2))


@pytest.mark.parametrize("N,K", [(8192, 64), (8197, 208), (14353, 48), (8200, 1040)])
@pytest.mark.parametrize("M", [9, 16, 17, 32, 33, 48, 49, 64])
def test_few_rows_of_wide_weights(dev, M, N, K):
    """Two tiles of weights a wave."""
    _case(t="wide", M=M, N=N, K=K)
    q, sx, (w,), (s,), b = _codes(M, N, K, 1)
    ref, tol = R.matmul(q, sx, w, s, b)
    R.check(mi_qmm.int8_matmul(q, w, s, x_scales=sx, bias=b, dtype=F32), ref, tol(F32), "y")
    ref, tol = R.matmul(q, sx, w, s)
    R.check(mi_qmm.int8_matmul(q, w, s, x_scales=sx), ref, tol(BF16), "bf16")


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("M,N,K", [(1840, 578, 7429), (1843, 577, 7440)])
def test_ranges_of_128_row_tiles(dev, M, N, K, t):
    """All blocks in one round: the kernel that asks the L2 for its lines ahead."""
    _case(t="ranges", M=M, N=N, K=K, type=t)
    q, sx, (w,), (s,), b = _codes(M, N, K, 1)
    ref, tol = R.matmul(q, sx, w, s, b.to(t))
    R.check(mi_qmm.int8_matmul(q, w, s, x_scales=sx, bias=b.to(t), dtype=t), ref, tol(t), "y")


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("M,N,K", [(57, 853, 208), (64, 130, 1040), (49, 36, 77)])
def test_gate_up_of_64_rows(dev, M, N, K, t):
    _case(t="gate + up", M=M, N=N, K=K, type=t)
    q, sx, w, s, _ = _codes(M, N, K, 2)
    got = mi_qmm.int8_gate_up_swiglu(q, w[0], s[0], w[1], s[1], x_scales=sx, dtype=t, save=True)
    r = R.gate_up(q, sx, w[0], s[0], w[1], s[1])
    # half a step past a type's largest value a rounding is infinite (fp16: 65520)
    top = float(torch.finfo(t).max)
    border = top + 2.0 ** math.floor(math.log2(top)) * torch.finfo(t).eps / 2
    for a, b, e in zip(got, r[:3], r[3:]):
        over = b.abs() > border
        assert ((b.abs() - border).abs() > e(t)).all()  # none lies next to the border
        R.check(a, torch.where(over, b.sign() * torch.inf, b), e(t), "gate + up")
