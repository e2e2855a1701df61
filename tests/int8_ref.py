"""The int8 operators in 64 bits, from their formulas, and how far a result may be from them.

u = 2^-24 is half a step of fp32; HALF[t] half a step of a type. Bounds are per value and count each
rounding on the way; `floor` is half of the type's smallest subnormal (fp16 outputs near zero)."""
import torch

U = 2.0 ** -24
HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
FLOOR = {torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25, torch.float32: 2.0 ** -150}
# fp16 parts of a scaled gradient and what they leave of it: half a step of 11 bits, and of what one
# part leaves where there are two. A row is scaled so that its largest value is 2^14 at least, and
# half of fp16's smallest subnormal, 2^-25, is then 2^-39 of that largest value.
PARTS = {torch.bfloat16: (1, 2.0 ** -11), torch.float16: (1, 2.0 ** -11), torch.float32: (2, 2.0 ** -22)}
SMALL = 2.0 ** -39


def quantize(x):
    """(codes, scales): the nearest integer to x / s, ties to even. The quotient of two 24-bit
    numbers is exact enough in 64 bits that a half-integer is met only where it is one."""
    s = (x.double().abs().amax(-1) / 127).float()
    q = torch.round(x.double() / s.double().unsqueeze(-1)).clamp(-127, 127)
    fine = torch.isfinite(s) & (s > 0)
    return torch.where(fine.unsqueeze(-1), q, torch.zeros_like(q)).to(torch.int8), s


def product(q, sx, w, sw):
    return (q.double() @ w.double().t()) * sx.double()[:, None] * sw.double()[None, :]


def check(y, ref, tol, what=""):
    """|y - ref| <= tol everywhere, not-a-numbers and infinities in the same places."""
    y, ref = y.double(), ref.double()
    fine = torch.isfinite(ref)
    assert torch.equal(torch.isnan(y), torch.isnan(ref)), f"{what}: NaN elsewhere"
    assert torch.equal(torch.isfinite(y), fine), f"{what}: infinite elsewhere"
    over = ((y - ref).abs() - tol)[fine]
    if over.numel():
        assert over.max().item() <= 0, f"{what}: {over.max().item():.3g} over the bound"


def matmul(q, sx, w, sw, bias=None):
    """(y, tolerance as a function of y's type): the sum is exact; its conversion, two products with
    scales and the sum with the bias round once each in fp32, then y."""
    p = product(q, sx, w, sw)
    y = p if bias is None else p + bias.double()
    return y, lambda t: 1.01 * (HALF[t] * y.abs() + U * (3 * p.abs() + y.abs())) + FLOOR[t]


def gate_up(q, sx, wg, sg, wu, su):
    """(y, gate, up, tolerance of y, of gate, of up). silu's relative condition number is at most
    1 + |g|: 3 roundings of g count that much; the exponential is off by 2 + 1.25 |g| (as in grads), and
    1 + e, the reciprocal (2) and the products add 8 at most. e^-g overflows below g = -88: 2^-120."""
    g, u = product(q, sx, wg, sg), product(q, sx, wu, su)
    y = g * torch.special.expit(g) * u
    rel = U * (3 * (1 + g.abs()) + 2 * (1 + g.abs()) + 3 + 5)

    def tol(t):
        return 1.01 * (HALF[t] + rel) * y.abs() + (g * u).abs() * 2.0 ** -120 + FLOOR[t]
    return (y, g, u, tol) + tuple(
        (lambda t, v=v: 1.01 * (HALF[t] + 3 * U) * v.abs() + FLOOR[t]) for v in (g, u))


def grads(dy, g, u):
    """(dgate, dup, tolerances before their rounding). s = 1 / (1 + 2^t), t = g log2(e): one ulp, 2 U, for
    the exponential and as much for the reciprocal, U for the sum; t is off by its rounding, U |t|,
    and by the constant's (0.23 U relative), which 2^t turns into 1.23 U |g|. 1 - s has the error of s
    as an absolute error."""
    dy, g, u = dy.double(), g.double(), u.double()
    s = torch.special.expit(g)
    dg, du = dy * u * (s + g * s * (1 - s)), dy * g * s
    es = U * (5 + 1.25 * g.abs())
    tg = (dy * u * s).abs() * ((1 + g.abs() * (1 - s)) * (es + 4 * U) + g.abs() * (s * es + 3 * U))
    tu = du.abs() * (es + 2 * U)
    # the reciprocal gives 0 for an s below 2^-126 (no subnormals): an absolute error of 2^-126 that
    # dgate multiplies by 1 + g (1 - s), at most 1 + |g|, and dup by g; twice that for the products
    # on the way, which may be subnormal too
    tiny = 2.0 ** -125
    return dg, du, 1.01 * tg + (dy * u).abs() * (1 + g.abs()) * tiny, 1.01 * tu + (dy * g).abs() * tiny


def through(a, ta, w, sw, t, top):
    """(sum_n a[m,n] sw[n] w[n,k], its tolerance before the output's rounding): the scaled value rounds
    once in fp32 and is cut to its fp16 parts (`top`: the row's largest); a sum of n terms is off by at
    most n steps (2 U) of the sum of their magnitudes, parts counted as terms, and the row's power of
    two is exact."""
    b = a * sw.double()[None, :]
    wd = w.double()
    parts, left = PARTS[t]
    n = a.shape[1] * parts
    mag = b.abs() @ wd.abs()
    err = (ta * sw.double()[None, :].abs()) @ wd.abs() + SMALL * top[:, None] * wd.abs().sum(0)
    return b @ wd, 1.01 * (mag * (left + U + 2 * U * n) + err)


def _top(*scaled):
    return torch.stack([v.abs().amax(1) for v in scaled]).amax(0)


def matmul_backward(dy, w, sw):
    t = dy.dtype
    dx, tol = through(dy.double(), torch.zeros_like(dy, dtype=torch.float64), w, sw, t, _top(dy.double() * sw.double()))
    return dx, 1.01 * HALF[t] * dx.abs() + tol + FLOOR[t]


def gate_up_backward(dy, g, u, wg, sg, wu, su):
    t = dy.dtype
    dg, du, tg, tu = grads(dy, g, u)
    top = _top(dg * sg.double(), du * su.double())
    a, ta = through(dg, tg, wg, sg, t, top)
    b, tb = through(du, tu, wu, su, t, top)
    dx = a + b
    out = lambda v, e: 1.01 * HALF[t] * v.abs() + e + FLOOR[t]
    # (the two banks are one sum of 2 N terms: each bound counts its own N once more)
    return (dx, dg, du), (out(dx, 2 * (ta + tb)), out(dg, tg), out(du, tu))
