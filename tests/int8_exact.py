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
