"""The int8 operators against their formulas in 64 bits (int8_ref.py), at the sizes, types and values
where they can go wrong."""
import ctypes

import pytest
import torch

import int8_ref as R
import mi_qmm
from mi_qmm import _lib as L

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
TYPES = [BF16, F16, F32]


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _weights(g, N, K):
    w = torch.randint(-127, 128, (N, K), device="cuda", generator=g, dtype=torch.int32).to(torch.int8)
    s = torch.rand(N, device="cuda", generator=g) * 1e-3 + 1e-5
    return w, s


def _x(g, M, K, t):
    return torch.randn(M, K, device="cuda", generator=g).to(t)


def _case(**kw):
    print("CASE", kw, flush=True)


# ---------------------------------------------------------------- quantization --
@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("M,K", [(1, 1), (1, 4096), (3, 8), (5, 63), (7, 64), (300, 72), (257, 520), (2, 1000),
                                 (259, 4096), (258, 5000), (260, 14336), (2, 14336), (1, 40000), (1, 131080),
                                 (258, 20008)])
def test_quantize(dev, M, K, t):
    _case(t="quantize", M=M, K=K, type=t)
    x = _x(_gen(M + K), M, K, t)
    q, s = mi_qmm.int8_quantize(x)
    rq, rs = R.quantize(x)
    assert torch.equal(s, rs) and torch.equal(q, rq)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("K", [16, 1000, 1001, 3000])
def test_quantize_borders(dev, K, t):
    """Values on and next to the border between two codes (scale 1: halves; scale an odd fraction),
    zero rows, infinities and NaN, the type's smallest and largest values."""
    h = torch.arange(K, device="cuda", dtype=torch.float64) % 255 - 127
    rows = [h + 0.5, h + 0.5 - 2.0 ** -7, (h + 0.5) * 3.0, torch.zeros_like(h), h, h, h,
            torch.full_like(h, float(torch.finfo(t).smallest_normal)), h * float(torch.finfo(t).tiny) / 64,
            torch.full_like(h, float(torch.finfo(t).max)), -h]
    x = torch.stack(rows).clamp(-float(torch.finfo(t).max), float(torch.finfo(t).max))
    x[:2].clamp_(-127, 127)
    x[:2, 0] = 127  # scale 1
    x = x.to(t)
    x[4, K // 2], x[5, K - 1], x[6, 0] = float("inf"), float("nan"), float("-inf")
    q, s = mi_qmm.int8_quantize(x)
    rq, rs = R.quantize(x)
    assert torch.equal(s.nan_to_num(-1), rs.nan_to_num(-1)) and torch.equal(q, rq)
    assert s[3] == 0 and not q[3].any() and torch.isnan(s[5]) and torch.isinf(s[4]) and not q[4:7].any()


def test_quantize_views_and_shapes(dev):
    x = _x(_gen(3), 6, 1024, BF16).view(2, 3, 1024)
    q, s = mi_qmm.int8_quantize(x)
    assert q.shape == (2, 3, 1024) and s.shape == (2, 3)
    off = torch.empty(6 * 1024 + 3, dtype=BF16, device="cuda")[3:].view(6, 1024)  # off 16 bytes
    off.copy_(x.view(6, 1024))
    q2, s2 = mi_qmm.int8_quantize(off)
    assert torch.equal(q.view(6, 1024), q2) and torch.equal(s.view(-1), s2)
    assert mi_qmm.int8_quantize(x[:0])[0].shape == (0, 3, 1024)


# ------------------------------------------------------------- forward products --
SHAPES = [(1, 1), (16, 16), (7, 33), (64, 64), (100, 208), (260, 1088), (130, 4096), (65, 77), (1111, 2000),
          (4096, 512)]
ROWS = [1, 2, 5, 15, 16, 17, 32, 33, 48, 64, 65, 100, 128, 129, 200, 257]


@pytest.mark.parametrize("N,K", SHAPES)
@pytest.mark.parametrize("M", ROWS)
def test_matmul_sizes(dev, M, N, K):
    _case(t="matmul", M=M, N=N, K=K)
    g = _gen(M * 31 + N)
    w, sw = _weights(g, N, K)
    x = _x(g, M, K, BF16)
    q, sx = R.quantize(x)
    ref, tol = R.matmul(q, sx, w, sw)
    y = mi_qmm.int8_matmul(x, w, sw)
    R.check(y, ref, tol(BF16), "float x")
    y2 = mi_qmm.int8_matmul(q, w, sw, x_scales=sx)
    assert torch.equal(y, y2)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("M,N,K", [(1, 260, 1024), (3, 100, 77), (40, 256, 320), (150, 136, 4096), (300, 520, 192)])
def test_matmul_types_and_bias(dev, M, N, K, t):
    _case(t="types", M=M, N=N, K=K, type=t)
    g = _gen(M + N)
    w, sw = _weights(g, N, K)
    x, b = _x(g, M, K, t), _x(g, 1, N, t)[0]
    q, sx = R.quantize(x)
    for out in TYPES:
        ref, tol = R.matmul(q, sx, w, sw, b.to(out))
        R.check(mi_qmm.int8_matmul(x, w, sw, bias=b.to(out), dtype=out), ref, tol(out), str(out))
    ref, tol = R.matmul(q, sx, w, sw)
    assert mi_qmm.int8_matmul(x, w, sw).dtype == t
    assert mi_qmm.int8_matmul(q, w, sw, x_scales=sx).dtype == BF16


@pytest.mark.parametrize("N,K", [(1, 1), (16, 64), (33, 208), (130, 77), (768, 2048), (2052, 512)])
@pytest.mark.parametrize("M", [1, 2, 16, 17, 33, 65, 100, 128, 129, 257])
def test_gate_up_sizes(dev, M, N, K):
    _case(t="gate_up", M=M, N=N, K=K)
    g = _gen(M * 7 + N)
    (wg, sg), (wu, su) = _weights(g, N, K), _weights(g, N, K)
    x = _x(g, M, K, BF16)
    q, sx = R.quantize(x)
    y, gate, up, ty, tg, tu = R.gate_up(q, sx, wg, sg, wu, su)
    o = mi_qmm.int8_gate_up_swiglu(x, wg, sg, wu, su, save=True)
    for a, b, t in zip(o, (y, gate, up), (ty, tg, tu)):
        R.check(a, b, t(BF16), "saved")
    assert torch.equal(mi_qmm.int8_gate_up_swiglu(x, wg, sg, wu, su), o[0])
    o2 = mi_qmm.int8_gate_up_swiglu(q, wg, sg, wu, su, x_scales=sx, save=True)
    assert all(torch.equal(a, b) for a, b in zip(o, o2))


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("M", [1, 20, 140])
def test_gate_up_types(dev, M, t):
    g = _gen(M)
    (wg, sg), (wu, su) = _weights(g, 200, 640), _weights(g, 200, 640)
    sg[3:20] *= 40  # gates beyond +-88, where e^-g leaves fp32
    x = _x(g, M, 640, t)
    q, sx = R.quantize(x)
    y, gate, up, ty, tg, tu = R.gate_up(q, sx, wg, sg, wu, su)
    for a, b, tol in zip(mi_qmm.int8_gate_up_swiglu(x, wg, sg, wu, su, save=True), (y, gate, up), (ty, tg, tu)):
        assert a.dtype == t
        R.check(a, b, tol(t), str(t))


@pytest.mark.parametrize("M", [1, 33, 130])
def test_largest_sums(dev, M):
    """131071 products of -128 by -128 (codes a caller made himself) stay below 2^31."""
    K = 131071
    x = torch.full((M, K), -128, dtype=torch.int8, device="cuda")
    w = torch.full((3, K), -128, dtype=torch.int8, device="cuda")
    w[1] = 127
    one = lambda n: torch.ones(n, device="cuda")
    y = mi_qmm.int8_matmul(x, w, one(3), x_scales=one(M), dtype=F32)
    want = torch.tensor([K * 16384.0, -K * 128.0 * 127.0, K * 16384.0], device="cuda", dtype=torch.float64).float()
    assert torch.equal(y, want.expand(M, 3))
    x16, w16 = x[:, :131056].contiguous(), w[:, :131056].contiguous()  # rows on 16 bytes
    y = mi_qmm.int8_matmul(x16, w16, one(3), x_scales=one(M), dtype=F32)
    want = torch.tensor([131056 * 16384.0, -131056 * 128.0 * 127.0, 131056 * 16384.0], device="cuda",
                        dtype=torch.float64).float()
    assert torch.equal(y, want.expand(M, 3))


@pytest.mark.parametrize("M", [2, 18, 40, 150])
@pytest.mark.parametrize("K", [96, 2048, 99])
def test_rows_are_independent(dev, M, K):
    """A row with an infinity or a NaN is NaN; a zero row gives the bias; the others keep their values.
    A NaN or infinite channel scale stays in its column."""
    g = _gen(M + K)
    w, sw = _weights(g, 72, K)
    x, b = _x(g, M, K, BF16), _x(g, 1, 72, BF16)[0]
    clean = mi_qmm.int8_matmul(x, w, sw, bias=b)
    xi, si = x.clone(), sw.clone()
    xi[0, 5], xi[M - 1, K - 1] = float("inf"), float("nan")
    si[41], si[7] = float("nan"), float("inf")
    y = mi_qmm.int8_matmul(xi, w, si, bias=b)
    assert torch.isnan(y[0]).all() and torch.isnan(y[M - 1]).all()
    cols = [n for n in range(72) if n not in (7, 41)]
    assert torch.equal(y[1:M - 1][:, cols], clean[1:M - 1][:, cols])
    assert torch.isnan(y[:, 41]).all() and not torch.isfinite(y[:, 7]).any()
    xi = x.clone()
    xi[M // 2] = 0
    y = mi_qmm.int8_matmul(xi, w, sw, bias=b)
    assert torch.equal(y[M // 2], b)
    assert not mi_qmm.int8_gate_up_swiglu(xi, w, sw, w, sw)[M // 2].any()


@pytest.mark.parametrize("M", [1, 20, 70, 300])
def test_unaligned_pointers(dev, M):
    """Views that start off 16 bytes give what aligned tensors give."""
    g = _gen(M)
    N, K = 132, 512
    w, sw = _weights(g, N, K)
    wu, su = _weights(g, N, K)
    x = _x(g, M, K, BF16)
    q, sx = mi_qmm.int8_quantize(x)

    def off(t, n):
        v = torch.empty(t.numel() + n, dtype=t.dtype, device="cuda")[n:].view(t.shape)
        v.copy_(t)
        return v
    y = mi_qmm.int8_matmul(x, w, sw)
    h = mi_qmm.int8_gate_up_swiglu(x, w, sw, wu, su)
    assert torch.equal(mi_qmm.int8_matmul(off(x, 1), w, sw), y)
    assert torch.equal(mi_qmm.int8_matmul(x, off(w, 3), off(sw, 1)), y)
    assert torch.equal(mi_qmm.int8_matmul(off(q, 5), w, sw, x_scales=off(sx, 1)), y)
    assert torch.equal(mi_qmm.int8_gate_up_swiglu(x, w, sw, off(wu, 1), su), h)
    dy = _x(g, M, N, BF16)
    dx = mi_qmm.int8_matmul_backward(dy, w, sw)
    R.check(mi_qmm.int8_matmul_backward(off(dy, 1), w, sw), *R.matmul_backward(dy, w, sw), "dy off")
    R.check(mi_qmm.int8_matmul_backward(dy, off(w, 3), sw), *R.matmul_backward(dy, w, sw), "w off")
    R.check(dx, *R.matmul_backward(dy, w, sw), "aligned")


# Sizes that reach every tile, its splits of K and the small tiles behind whole rounds of big ones; K ends
# inside a step (a multiple of 16 only), rows and columns inside tiles.
@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("M,N,K", [(1100, 9000, 2064), (2600, 7700, 2064), (2600, 7701, 1040), (600, 5002, 2064),
                                   (1300, 2000, 1040), (300, 1000, 4112), (600, 1001, 8208), (150, 700, 8208),
                                   (129, 24, 16400), (257, 4104, 16), (129, 24301, 64), (3615, 38, 9232), (3588, 40, 10112),
                                   (165, 22405, 1296), (141, 4469, 9792), (1784, 16822, 272), (6205, 6142, 608),
                                   (457, 17435, 12448), (146, 12147, 9600)])
def test_matmul_tiles(dev, M, N, K, t):
    _case(t="matmul_tiles", M=M, N=N, K=K, type=t)
    g = _gen(M + N)
    w, sw = _weights(g, N, K)
    x = _x(g, M, K, t)
    q, sx = mi_qmm.int8_quantize(x)
    b = _x(g, 1, N, t)[0]
    ref, tol = R.matmul(q, sx, w, sw, b)
    y = mi_qmm.int8_matmul(x, w, sw, bias=b)
    R.check(y, ref, tol(t), "y")
    assert torch.equal(y, mi_qmm.int8_matmul(x, w, sw, bias=b))


@pytest.mark.parametrize("t,save", [(BF16, True), (F16, False), (F32, True)])
@pytest.mark.parametrize("M,N,K", [(1100, 4500, 2064), (1300, 13000, 1040), (600, 2501, 2064), (300, 1000, 4112),
                                   (600, 1000, 8208), (150, 350, 8208), (700, 10000, 528), (129, 35, 64), (135, 12137, 64),
                                   (1673, 257, 8064), (158, 11369, 1184), (139, 3614, 6048), (464, 30050, 272),
                                   (7836, 1312, 784), (135, 17529, 10144), (136, 5754, 9472)])
def test_gate_up_tiles(dev, M, N, K, t, save):
    _case(t="gate_up_tiles", M=M, N=N, K=K, type=t)
    g = _gen(M + N)
    (wg, sg), (wu, su) = _weights(g, N, K), _weights(g, N, K)
    x = _x(g, M, K, t)
    q, sx = mi_qmm.int8_quantize(x)
    y, gate, up, ty, tg, tu = R.gate_up(q, sx, wg, sg, wu, su)
    o = mi_qmm.int8_gate_up_swiglu(x, wg, sg, wu, su, save=save)
    for a, b, tol in zip(o if save else (o,), (y, gate, up), (ty, tg, tu)):
        R.check(a, b, tol(t), "saved")


# ------------------------------------------------------------------- gradients --
@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("M,K,N", [(520, 32992, 130), (1100, 9008, 2050), (2600, 7696, 1026), (600, 5008, 2050),
                                   (130, 5008, 2050), (300, 1008, 4100), (600, 1008, 8200), (70, 528, 8200),
                                   (257, 16, 2049), (204, 32, 8282), (2621, 144, 5040), (3313, 288, 12279),
                                   (520, 16512, 1030), (3313, 8208, 260)])
def test_matmul_backward_tiles(dev, M, K, N, t):
    _case(t="matmul_bwd_tiles", M=M, N=N, K=K, type=t)
    g = _gen(M + N)
    w, sw = _weights(g, N, K)
    dy = _x(g, M, N, t)
    dx = mi_qmm.int8_matmul_backward(dy, w, sw)
    R.check(dx, *R.matmul_backward(dy, w, sw), "dx")
    assert torch.equal(dx, mi_qmm.int8_matmul_backward(dy, w, sw))


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("M,K,N", [(1100, 9008, 520), (2600, 7696, 514), (130, 1008, 2050), (300, 2000, 14336)])
def test_gate_up_backward_tiles(dev, M, K, N, t):
    _case(t="gate_up_bwd_tiles", M=M, N=N, K=K, type=t)
    g = _gen(M + N)
    (wg, sg), (wu, su) = _weights(g, N, K), _weights(g, N, K)
    dy, gate, up = _x(g, M, N, t), _x(g, M, N, t) * 2, _x(g, M, N, t)
    ref, tol = R.gate_up_backward(dy, gate, up, wg, sg, wu, su)
    for a, r, e, what in zip(mi_qmm.int8_gate_up_swiglu_backward(dy, gate, up, wg, sg, wu, su), ref, tol,
                             ("dx", "dgate", "dup")):
        R.check(a, r, e, what)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("N,K", [(1, 1), (16, 64), (33, 208), (130, 77), (64, 4096), (1536, 520), (2052, 132)])
@pytest.mark.parametrize("M", [1, 2, 17, 64, 65, 129, 300])
def test_matmul_backward(dev, M, N, K, t):
    _case(t="matmul_bwd", M=M, N=N, K=K, type=t)
    g = _gen(M + N + K)
    w, sw = _weights(g, N, K)
    dy = _x(g, M, N, t)
    R.check(mi_qmm.int8_matmul_backward(dy, w, sw), *R.matmul_backward(dy, w, sw), "dx")


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("N,K", [(1, 1), (16, 64), (33, 208), (130, 77), (768, 512), (2052, 132)])
@pytest.mark.parametrize("M", [1, 3, 64, 129, 300])
def test_gate_up_backward(dev, M, N, K, t):
    _case(t="gate_up_bwd", M=M, N=N, K=K, type=t)
    g = _gen(M + N + K)
    (wg, sg), (wu, su) = _weights(g, N, K), _weights(g, N, K)
    dy, gate, up = _x(g, M, N, t), _x(g, M, N, t) * 2, _x(g, M, N, t)
    gate.view(-1)[::7] *= 60  # saturated on both sides
    ref, tol = R.gate_up_backward(dy, gate, up, wg, sg, wu, su)
    for a, r, e, what in zip(mi_qmm.int8_gate_up_swiglu_backward(dy, gate, up, wg, sg, wu, su), ref, tol,
                             ("dx", "dgate", "dup")):
        assert a.dtype == t
        R.check(a, r, e, what)


def test_gradients_by_differences(dev):
    """The formulas' gradients against central differences of the forward formula in 64 bits, on
    activations before rounding: step 1e-4 leaves at most 1e-7 of truncation on values of order 1."""
    g = _gen(5)
    M, N, K = 5, 24, 40
    (wg, sg), (wu, su), (wd, sd) = _weights(g, N, K), _weights(g, N, K), _weights(g, 16, N)
    f64 = lambda w, s: w.double() * s.double()[:, None]
    x = _x(g, M, K, F32)
    dy = _x(g, M, 16, F32)

    def loss(v):
        a, b = v @ f64(wg, sg).t(), v @ f64(wu, su).t()
        return ((a * torch.special.expit(a) * b) @ f64(wd, sd).t() * dy.double()).sum()
    gate, up = (x.double() @ f64(wg, sg).t()).float(), (x.double() @ f64(wu, su).t()).float()
    dh = mi_qmm.int8_matmul_backward(dy, wd, sd)
    dx, _, _ = mi_qmm.int8_gate_up_swiglu_backward(dh, gate, up, wg, sg, wu, su)
    for m, k in ((0, 0), (2, 17), (4, 39)):
        e = torch.zeros(M, K, device="cuda", dtype=torch.float64)
        e[m, k] = 1e-4
        d = (loss(x.double() + e) - loss(x.double() - e)) / 2e-4
        # fp32 operands: gate and up rounded (2^-24 of values of order 1), sums of 24 and 40 terms
        assert abs(d.item() - dx[m, k].item()) <= 1e-6 * dx.abs().max().item() + 1e-9


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("M", [3, 130])
def test_gradients_with_infinite_values(dev, M, t):
    """An infinity or NaN in a gradient stays in its row; the others keep their values."""
    g = _gen(M)
    w, sw = _weights(g, 130, 200)
    w[5] = w[5].abs().clamp(min=1)
    dy = _x(g, M, 130, t)
    clean = mi_qmm.int8_matmul_backward(dy, w, sw)
    bad = dy.clone()
    bad[0, 5], bad[M - 1, 129] = float("inf"), float("nan")
    dx = mi_qmm.int8_matmul_backward(bad, w, sw)
    assert torch.equal(dx[1:M - 1], clean[1:M - 1])
    assert torch.isnan(dx[M - 1]).all() and not torch.isfinite(dx[0]).any()


@pytest.mark.parametrize("t,big", [(BF16, 1e30), (F16, 3e4), (F32, 1e30)])
def test_gradients_beside_an_infinity(dev, t, big):
    """Finite values beside an infinity, larger than fp16 holds, stay finite: the sum is infinite where
    the infinity's code is not 0, NaN where it is, as the formula has it."""
    w = torch.tensor([[1, -2, 0, 5], [3, 4, 5, -6], [-7, 8, 9, 10]], dtype=torch.int8, device="cuda").repeat(1, 8)
    sw = torch.ones(3, device="cuda")
    dy = torch.tensor([[float("inf"), -big, big], [1.0, big, -big], [2.0 ** -20, 0.0, 1.0]], device="cuda").to(t)
    dx = mi_qmm.int8_matmul_backward(dy, w, sw)
    assert torch.isnan(dx[0, 2]) and torch.isinf(dx[0, [0, 1, 3]]).all() and dx[0, 1] < 0 < dx[0, 0]
    ref, tol = R.matmul_backward(dy[1:], w, sw)
    # 3e4 (1 * 0 + 3 + 7) is 3e5: past fp16's largest value and half a step (65520) a rounding is infinite
    ref = torch.where(ref.abs() - tol > torch.finfo(t).max * (1 + torch.finfo(t).eps / 4), ref.sign() * torch.inf, ref)
    R.check(dx[1:], ref, tol, "finite rows")


def test_offsets_past_31_bits(dev):
    """More than 2^31 values of x and of y: the last rows against the same rows alone."""
    g = _gen(9)
    M, K, N = 70001, 31008, 64
    x = torch.randn(M, K, device="cuda", generator=g, dtype=BF16)
    q, s = mi_qmm.int8_quantize(x)
    ql, sl = R.quantize(x[-5:])
    assert torch.equal(q[-5:], ql) and torch.equal(s[-5:], sl)
    w, sw = _weights(g, N, K)
    y = mi_qmm.int8_matmul(q, w, sw, x_scales=s)
    ref, tol = R.matmul(ql, sl, w, sw)
    R.check(y[-5:], ref, tol(BF16), "rows far into x")
    del y, x
    w, sw = _weights(g, K, N)
    x = _x(g, M, N, BF16)
    y = mi_qmm.int8_matmul(x, w, sw)
    qx, sx = R.quantize(x[-5:])
    ref, tol = R.matmul(qx, sx, w, sw)
    R.check(y[-5:], ref, tol(BF16), "rows far into y")
    dx = mi_qmm.int8_matmul_backward(y, w, sw)
    R.check(dx[-5:], *R.matmul_backward(y[-5:], w, sw), "rows far into dy")
    del dx, y
    dx = mi_qmm.int8_matmul_backward(x, w.t().contiguous(), torch.ones(N, device="cuda"))
    R.check(dx[-5:], *R.matmul_backward(x[-5:], w.t().contiguous(), torch.ones(N, device="cuda")), "rows far into dx")


# ------------------------------------------------- as they are used, and around --
def _block(g, hidden, inter):
    mk = lambda n, k: mi_qmm.int8_quantize(torch.randn(n, k, device="cuda", generator=g) * 0.05)
    return mk(inter, hidden), mk(inter, hidden), mk(hidden, inter)


@pytest.mark.parametrize("M", [1, 7, 160])
def test_feed_forward_block(dev, M):
    """Quantized tokens through gate + up and the down projection, and the gradient back: each step
    against the formula on what it was given."""
    g = _gen(M)
    (wg, sg), (wu, su), (wd, sd) = _block(g, 256, 704)
    x = _x(g, M, 256, BF16)
    q, sx = mi_qmm.int8_quantize(x)
    h, gate, up = mi_qmm.int8_gate_up_swiglu(q, wg, sg, wu, su, x_scales=sx, dtype=BF16, save=True)
    R.check(h, (r := R.gate_up(q, sx, wg, sg, wu, su))[0], r[3](BF16), "h")
    y = mi_qmm.int8_matmul(h, wd, sd)
    hq, hs = R.quantize(h)
    ref, tol = R.matmul(hq, hs, wd, sd)
    R.check(y, ref, tol(BF16), "y")
    dy = _x(g, M, 256, BF16)
    dh = mi_qmm.int8_matmul_backward(dy, wd, sd)
    R.check(dh, *R.matmul_backward(dy, wd, sd), "dh")
    got = mi_qmm.int8_gate_up_swiglu_backward(dh, gate, up, wg, sg, wu, su)
    for a, b, t in zip(got, *R.gate_up_backward(dh, gate, up, wg, sg, wu, su)):
        R.check(a, b, t, "back")


def _run_block(x, W, dy):
    (wg, sg), (wu, su), (wd, sd) = W
    h, gate, up = mi_qmm.int8_gate_up_swiglu(x, wg, sg, wu, su, save=True)
    y = mi_qmm.int8_matmul(h, wd, sd)
    dh = mi_qmm.int8_matmul_backward(dy, wd, sd)
    return (y,) + mi_qmm.int8_gate_up_swiglu_backward(dh, gate, up, wg, sg, wu, su)


@pytest.mark.parametrize("M", [1, 40, 200])
def test_graphs(dev, M):
    """Two captured graphs of the block on two streams, replayed in turn and at the same time, with
    eager calls between, give the eager results every time."""
    g = _gen(M)
    W = _block(g, 256, 704)
    xs = [_x(g, M, 256, BF16) for _ in range(2)]
    dys = [_x(g, M, 256, BF16) for _ in range(2)]
    want = [_run_block(xs[i], W, dys[i]) for i in range(2)]
    torch.cuda.synchronize()
    graphs, outs, streams = [], [], [torch.cuda.Stream(), torch.cuda.Stream()]
    for i in range(2):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr, stream=streams[i]):
            outs.append(_run_block(xs[i], W, dys[i]))
        graphs.append(gr)
    for turn in range(4):
        for i in range(2):
            for o in outs[i]:
                o.zero_()
        torch.cuda.synchronize()
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                graphs[i].replay()
        eager = _run_block(xs[0], W, dys[0])
        torch.cuda.synchronize()
        for i in range(2):
            assert all(torch.equal(a, b) for a, b in zip(outs[i], want[i])), (turn, i)
        assert all(torch.equal(a, b) for a, b in zip(eager, want[0]))


@pytest.mark.parametrize("M,N,K", [(1, 100, 64), (17, 36, 128), (70, 66, 96), (130, 258, 320)])
def test_nothing_written_behind_the_outputs(dev, M, N, K):
    """Through the C ABI into larger buffers: what lies behind the last row stays."""
    g = _gen(1)
    w, sw = _weights(g, N, K)
    x = _x(g, M, K, BF16)
    lib, P = L.lib(), lambda t: ctypes.c_void_p(t.data_ptr())
    ws = torch.empty(lib.mi_int8_forward_workspace(M, N, K, 2, L.DT_BFLOAT16) + 256, dtype=torch.uint8, device="cuda")
    s = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
    bufs = [torch.full((M * N + 512,), 77.0, dtype=BF16, device="cuda") for _ in range(3)]
    need = ws.numel() - 256
    ws[need:] = 99
    L.check(lib.mi_int8_gate_up_swiglu(*[P(b) for b in bufs], P(x), None, P(w), P(sw), P(w), P(sw), M, N, K,
                                       L.DT_BFLOAT16, L.DT_BFLOAT16, P(ws), need, s))
    assert all((b[M * N:] == 77).all() for b in bufs) and (ws[need:] == 99).all()
    y = mi_qmm.int8_gate_up_swiglu(x, w, sw, w, sw)
    assert torch.equal(bufs[0][:M * N].view(M, N), y)
    dx = torch.full((M * K + 512,), 77.0, dtype=BF16, device="cuda")
    need = lib.mi_int8_backward_workspace(M, N, K, 1, L.DT_BFLOAT16)
    ws = torch.full((need + 256,), 99, dtype=torch.uint8, device="cuda")
    dy = _x(g, M, N, BF16)
    L.check(lib.mi_int8_matmul_backward(P(dx), P(dy), P(w), P(sw), M, N, K, L.DT_BFLOAT16, P(ws), need, s))
    assert (dx[M * K:] == 77).all() and (ws[need:] == 99).all()
    assert torch.equal(dx[:M * K].view(M, K), mi_qmm.int8_matmul_backward(dy, w, sw))


def test_leading_dimensions_and_empty(dev):
    g = _gen(2)
    w, sw = _weights(g, 48, 64)
    x = _x(g, 6, 64, BF16)
    y = mi_qmm.int8_matmul(x, w, sw)
    assert torch.equal(mi_qmm.int8_matmul(x.view(2, 3, 64), w, sw), y.view(2, 3, 48))
    assert torch.equal(mi_qmm.int8_matmul(x[0], w, sw), y[0])
    assert mi_qmm.int8_matmul(x[:0], w, sw).shape == (0, 48)
    assert mi_qmm.int8_matmul(x, w[:0], sw[:0]).shape == (6, 0)
    assert mi_qmm.int8_gate_up_swiglu(x[:0], w, sw, w, sw).shape == (0, 48)
    assert mi_qmm.int8_matmul_backward(y[:0], w, sw).shape == (0, 64)
    with pytest.raises(mi_qmm.MiError):
        mi_qmm.int8_matmul_backward(y[:, :0].contiguous(), w[:0], sw[:0])
    for call in (lambda: mi_qmm.int8_matmul(x.new_empty(2, 3, 0), w[:, :0].contiguous(), sw),
                 lambda: mi_qmm.int8_matmul_backward(y.new_empty(2, 3, 0), w[:0], sw[:0]),
                 lambda: mi_qmm.int8_quantize(x.new_empty(2, 0))):
        with pytest.raises(mi_qmm.MiError):
            call()
    assert mi_qmm.int8_matmul(x.new_empty(2, 0, 64), w, sw).shape == (2, 0, 48)
    assert mi_qmm.int8_matmul_backward(y.new_empty(0, 3, 48), w, sw).shape == (0, 3, 64)
    q, s = mi_qmm.int8_quantize(x.view(2, 3, 64))
    assert q.shape == (2, 3, 64) and s.shape == (2, 3) and mi_qmm.int8_quantize(x[0])[1].shape == ()
    assert mi_qmm.int8_quantize(x.new_empty(2, 0, 64))[1].shape == (2, 0)
    z = mi_qmm.int8_gate_up_swiglu(x.view(2, 3, 64), w, sw, w, sw, save=True)
    dh = mi_qmm.int8_gate_up_swiglu_backward(z[0], z[1], z[2], w, sw, w, sw)
    assert all(t.shape == (2, 3, 48) and t.is_contiguous() for t in z) and dh[0].shape == (2, 3, 64)


def test_refusals_on_device(dev):
    g = _gen(2)
    w, sw = _weights(g, 48, 64)
    x = _x(g, 6, 64, BF16)
    q, sx = mi_qmm.int8_quantize(x)
    for call in (lambda: mi_qmm.int8_matmul(x.t(), w, sw), lambda: mi_qmm.int8_matmul(x[:, ::2], w[:, :32], sw),
                 lambda: mi_qmm.int8_matmul(x[:, :32].contiguous(), w, sw), lambda: mi_qmm.int8_matmul(q, w, sw),
                 lambda: mi_qmm.int8_matmul(x, w, sw, x_scales=sx), lambda: mi_qmm.int8_matmul(x, w, sw[:40]),
                 lambda: mi_qmm.int8_matmul(x, w, sw.half()), lambda: mi_qmm.int8_matmul(x.double(), w, sw),
                 lambda: mi_qmm.int8_matmul(q, w, sw, x_scales=sx[:3]), lambda: mi_qmm.int8_matmul(x, w.cpu(), sw),
                 lambda: mi_qmm.int8_matmul(x, w, sw, bias=sw), lambda: mi_qmm.int8_matmul(x, w, sw, dtype=torch.int8),
                 lambda: mi_qmm.int8_gate_up_swiglu(x, w, sw, w[:40], sw[:40]),
                 lambda: mi_qmm.int8_matmul_backward(x, w, sw), lambda: mi_qmm.int8_matmul_backward(q, w, sw),
                 lambda: mi_qmm.int8_gate_up_swiglu_backward(x[:, :48].contiguous(), x, x, w, sw, w, sw)):
        with pytest.raises(mi_qmm.MiError):
            call()
