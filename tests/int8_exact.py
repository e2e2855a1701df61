"""Data on which the int8 gradients have one right answer, and how far a result may be where they do not.

The bounds of int8_ref.py charge every rounding of a long sum at its worst, so that at thousands of terms a lost
one passes. Here sums are exact in fp32 in any order (integers below 2^24, checked), or have few terms.
U = 2^-24 is half a step of fp32."""
import torch

U = 2.0 ** -24
F32 = torch.float32
# of the types that a gradient comes in: half a step, and half of the smallest subnormal
HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
FLOOR = {torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25, torch.float32: 2.0 ** -150}


def gen(seed, device):
    return torch.Generator(device=device).manual_seed(seed)


def _ints(g, shape, lo, hi, device):
    return torch.randint(lo, hi + 1, shape, generator=g, device=device, dtype=torch.int32)


def _powers(g, n, lo, hi, device):
    return torch.exp2(_ints(g, (n,), lo, hi, device).float())


def rounded(v, t):
    """An exact fp32 value (given in 64 bits) as t."""
    assert torch.equal(v.float().double(), v)
    return v.float().to(t)


# ------------------------------------------------------------ sums that are exact --
def _dense(g, M, N, K, device):
    """Three bits a value, every code: each term counts."""
    dy = _ints(g, (M, N), -3, 3, device).float()
    w = [_ints(g, (N, K), -127, 127, device).to(torch.int8) for _ in range(2)]
    return dy, w, [_powers(g, N, -9, -8, device) for _ in range(2)]


def _sparse(g, M, N, K, t, banks, device):
    """Values and scales whose products have 20 bits (24 of one fp32 value), few codes a column: each bit counts."""
    top, s_top = {torch.bfloat16: (255, 4095), torch.float16: (2047, 511), torch.float32: ((1 << 24) - 1, 1)}[t]
    dy = _ints(g, (M, N), -top, top, device).float()
    s = _ints(g, (N,), s_top // 2 + 1, s_top, device).float() * 2.0 ** -9
    w = [torch.zeros(N, K, dtype=torch.int8, device=device) for _ in range(banks)]
    k = torch.arange(K, device=device)
    terms = 1 if t == F32 else 4
    for b in range(banks):
        for j in range(terms):
            c = _ints(g, (K,), 1, 4 // banks if terms > 1 else 1, device) * (1 - 2 * _ints(g, (K,), 0, 1, device))
            if terms == 1:
                c = c * (k % banks == b)
            w[b][(N - 1 - k - j * (N // 4)) % N, k] += c.to(torch.int8)  # (rows of a column meet where N < 4: c adds up)
    return dy, w, [s] * banks


def product_case(M, N, K, t, dense, device, seed=0):
    """(dy, w, scales)"""
    g = gen(seed + M + 3 * N + 7 * K, device)
    dy, w, s = _dense(g, M, N, K, device) if dense else _sparse(g, M, N, K, t, 1, device)
    return dy.to(t), w[0], s[0]


def gated_case(M, N, K, t, dense, device, seed=0):
    """(dy, gate, up, w, scales) of two banks. gate = 64, where the sigmoid is 1 in fp32 and its derivative nothing
    beside 1, so that dgate = dy up and dup = 64 dy: integers again."""
    g = gen(seed + M + 3 * N + 7 * K, device)
    dy, w, s = _dense(g, M, N, K, device) if dense else _sparse(g, M, N, K, t, 2, device)
    up = _powers(g, M * N, 0, 1 if dense else 0, device).view(M, N)
    return dy.to(t), torch.full((M, N), 64.0, device=device).to(t), up.to(t), w, [s[0], s[1] / 64]


def exact_sum(a, w):
    """sum over the banks of a @ w (a: the scaled gradients) in 64 bits, where every partial sum is a whole multiple of
    2^-9 below 2^24 of them."""
    mag = sum(v.double().abs() @ c.double().abs() for v, c in zip(a, w))
    assert mag.max().item() < 2.0 ** 15
    assert all(torch.equal(v * 512, (v * 512).round()) for v in a)
    return sum(v.double() @ c.double() for v, c in zip(a, w))


def scaled(d, s):
    return [x.double() * y.double() for x, y in zip(d, s)]


def rounded(v, t):
    """Values that fp32 holds, in 64 bits, as t."""
    assert torch.equal(v.float().double(), v)
    return v.float().to(t)


# ------------------------------------------------------- what a value keeps of its bits --
def wide_case(M, N, span, device, seed=0):
    """fp32 rows whose values have 24 bits and lie between the row's largest and 2^-span of it; one code a column, a
    power of two, so that dx = dy w has dy's bits."""
    g = gen(seed + M + N, device)
    m = _ints(g, (M, N), 1 << 23, (1 << 24) - 1, device).float()
    e = _ints(g, (M, N), 0, span, device)
    e[:, 0] = 0
    dy = m * torch.exp2(-23.0 - e.float()) * (1 - 2 * _ints(g, (M, N), 0, 1, device)).float()
    dy[:, 0] = m[:, 0].abs() * 2.0 ** -23
    dy = dy * _powers(g, M, -30, 30, device)[:, None]
    w = torch.diag(torch.exp2((torch.arange(N, device=device) % 7).float()) * (1 - 2 * (torch.arange(N, device=device) % 2))).to(torch.int8)
    return dy, w, torch.ones(N, device=device)


def cancelling_case(M, N, t, device, seed=0):
    """Columns that take the difference of two products dy s with equal dy and scales 2^-9 apart or less: what each
    product lost counts 2^9 times as much. (dx, bound)."""
    g = gen(seed + M + N, device)
    dy = torch.randn(M, N // 2, generator=g, device=device).to(t).repeat_interleave(2, 1)
    s = torch.rand(N // 2, generator=g, device=device) + 1
    s = torch.stack([s, s * (1 + 2.0 ** -9 * torch.rand(N // 2, generator=g, device=device))], 1).view(-1)
    c = _ints(g, (N // 2,), 1, 127, device).to(torch.int8)
    w = torch.zeros(N, N // 2, dtype=torch.int8, device=device)
    k = torch.arange(N // 2, device=device)
    w[2 * k, k], w[2 * k + 1, k] = c, -c
    return dy.contiguous(), w, s


def cancelling_sum(dy, w, s, left):
    """(dx, bound): each product rounds once in fp32 and loses `left` of itself on its way into the sum; the sum has
    at most six partial products, one step (2 U) of all their magnitudes each."""
    a = dy.double() * s.double()
    mag = a.abs() @ w.double().abs()
    dx = a @ w.double()
    return dx, 1.01 * (HALF[dy.dtype] * dx.abs() + mag * (left + U + 12 * U)) + FLOOR[dy.dtype]


# ---------------------------------------------------------------- the fp32 sigmoid --
# s = 1 / (1 + e) or e / (1 + e), e = exp(-|g|) to one ulp (2 U), the sum, the quotient and the product U each:
# 6 U at most. An e below 2^-126 is off by a subnormal step at most.
SIG = 6 * U
STEP = 2.0 ** -148


def silu_case(device):
    """Codes whose gate is a b / 128 exactly, -126 .. 126, and whose up is a power of two up to 2^100."""
    a = torch.arange(-127, 128, device=device)
    b = torch.arange(1, 128, 2, device=device)
    x = torch.zeros(a.numel(), 16, dtype=torch.int8, device=device)
    x[:, 0], x[:, 1] = a.to(torch.int8), 1
    wg = torch.zeros(b.numel(), 16, dtype=torch.int8, device=device)
    wu = wg.clone()
    wg[:, 0], wu[:, 1] = b.to(torch.int8), 1
    sg = torch.full((b.numel(),), 2.0 ** -7, device=device)
    su = torch.exp2((b % 4).float() / 3 * 100).clamp(max=2.0 ** 100)
    su = torch.exp2(torch.log2(su).round())
    return x, torch.ones(a.numel(), device=device), wg, sg, wu, su


def silu(x, wg, sg, wu, su):
    """(y, bound) of silu_case: two products more than the sigmoid."""
    g, u = (x.double() @ w.double().t() * s.double() for w, s in ((wg, sg), (wu, su)))
    y = g * torch.special.expit(g) * u
    return y, 1.01 * (SIG + 2 * U) * y.abs() + (g * u).abs() * STEP + FLOOR[F32]


def dsilu(dy, g, u):
    """(dgate, dup, bounds): s and 1 - s to SIG each; dgate = ((dy u) s) (1 + g (1 - s)). Where (dy u) s is
    subnormal it rounds by half a step, 2^-150, which the last factor multiplies."""
    dy, g, u = dy.double(), g.double(), u.double()
    s, c = torch.special.expit(g), torch.special.expit(-g)
    f = 1 + g * c
    dg, du = dy * u * s * f, dy * g * s
    tg = (dy * u * s).abs() * ((g * c).abs() * (SIG + U) + f.abs() * (SIG + 4 * U))
    return (dg, du, 1.01 * tg + (dy * u).abs() * (1 + g.abs()) * STEP + (1 + f.abs()) * FLOOR[F32],
            1.01 * du.abs() * (SIG + 3 * U) + (dy * g).abs() * STEP + FLOOR[F32])
