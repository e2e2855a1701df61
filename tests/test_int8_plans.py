"""The kernels that the sizes of the int8 GPU tests take, by the library's own plans (tests/cpp/int8_plan.cpp): a
change of a plan that leaves a kernel without a test fails here."""
import os
import random
import subprocess

import pytest

import test_gpu_int8 as T
import test_gpu_int8_exact as E
from mi_qmm import _lib as L

BIN = os.path.join(os.path.dirname(os.path.abspath(__file__)), "cpp", "_build", "int8_plan")
FEW = {1: [(x, w) for w in (1, 2) for x in (1, 2, 3, 4)] + [(6, 1), (8, 1)], 2: [(x, 1) for x in (1, 2, 3, 4, 6, 8)]}
TILES = ("256 256", "128 256", "128 128", "64 128")
RINGS_OF_TWO = ("256 256", "128 128")


def plans(lines):
    """The launches of each call: (way, banks, bytes of x's or a gradient's type, M, N, K)."""
    if not os.path.exists(BIN):
        pytest.fail(f"{BIN} not built (run __graft_entry__.build())")
    r = subprocess.run([BIN], input="\n".join(" ".join(map(str, l)) for l in lines) + "\n", capture_output=True,
                       text=True, timeout=60, check=True)
    return [set(o.split(": ")[1].split(", ")) for o in r.stdout.splitlines()]


def sizes(test):
    """Every combination of a test's parameters, by name."""
    out = [{}]
    for m in test.pytestmark:
        if m.name == "parametrize":
            names = m.args[0].split(",")
            values = [v if len(names) > 1 else (v,) for v in m.args[1]]
            out = [dict(o, **dict(zip(names, v))) for o in out for v in values]
    return out


def reached(way, banks, tests, size):
    lines = [(way, banks, size, c.get("M", 1), c.get("N", 100), c["K"]) for t in tests for c in sizes(t)]
    return set().union(*plans(lines))


def forward_kernels(banks):
    tiles = {f"tile {t} {s}{a}" for t in TILES for s in ("whole", "split")
             for a in (("", " ahead") if t in RINGS_OF_TWO else ("",))}
    return tiles | {"tile 128 256 tail", "token 1", "token 4"} | {f"few {x} {w}" for x, w in FEW[banks]}


BACKWARD = {f"tile {t} {s}" for t in TILES for s in ("whole", "split")} | {"tile 128 256 tail"}
FORWARD_TESTS = {
    1: ((T.test_matmul_sizes, 2), (T.test_matmul_tiles, 2), (E.test_long_float_token, 2), (E.test_few_rows_of_wide_weights, 0),
        (E.test_ranges_of_128_row_tiles, 0)),
    2: ((T.test_gate_up_sizes, 2), (T.test_gate_up_tiles, 2), (E.test_long_float_token, 2), (E.test_gate_up_of_64_rows, 0))}


@pytest.mark.parametrize("banks", [1, 2])
def test_every_forward_kernel_is_tested(banks):
    got = set().union(*(reached("f", banks, [t], size) for t, size in FORWARD_TESTS[banks]))
    assert got == forward_kernels(banks)


@pytest.mark.parametrize("size", [2, 4])
@pytest.mark.parametrize("banks,test", [(1, E.test_exact_product_gradients), (2, E.test_exact_gated_gradients)])
def test_every_gradient_kernel_is_tested(banks, test, size):
    assert reached("b", banks, [test], size) == BACKWARD


def test_no_size_takes_another_kernel():
    r = random.Random(1)
    n = lambda top: int(top ** r.random())
    for banks in (1, 2):
        f = [("f", banks, r.choice((0, 2, 4)), n(20000), n(40000), n(40000)) for _ in range(10000)]
        assert set().union(*plans(f)) <= forward_kernels(banks)
        b = [("b", banks, r.choice((2, 4)), n(20000), n(40000), n(40000)) for _ in range(10000)]
        assert set().union(*plans(b)) <= BACKWARD


@pytest.mark.parametrize("banks", [1, 2])
@pytest.mark.parametrize("dtype,size,parts", [(L.DT_BFLOAT16, 2, 2), (L.DT_FLOAT16, 2, 2), (L.DT_FLOAT32, 4, 3)])
def test_the_calls_take_these_plans(banks, dtype, size, parts):
    """A split product's sums show in the workspace that the call asks for."""
    up = lambda v, to: -(-v // to) * to
    cases = sorted({(c["M"], c["N"], c["K"]) for c in sizes(E.test_exact_product_gradients)})
    for (M, N, K), plan in zip(cases, plans([("b", banks, size) + c for c in cases])):
        rest = up(banks * parts * M * up(N, 64) * 2, 256) + up(4 * M, 256)
        rest += banks * up(N * up(K, 16), 256) if K % 16 else 0
        sums = L.lib().mi_int8_backward_workspace(M, N, K, banks, dtype) - rest
        assert (sums > 0) == any("split" in p for p in plan) and sums % (4 * M * up(K, 16)) == 0 <= sums
