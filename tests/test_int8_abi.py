"""What the int8 entry points refuse, without a GPU: every bad call ends in its code and a message before
the device is touched. And the 64-bit formulas that the GPU tests compare with."""
import ctypes

import pytest
import torch

import int8_ref as R
import mi_qmm
from mi_qmm import _lib as L

P = ctypes.c_void_p


def _forward(fn="mi_int8_matmul", **kw):
    a = dict(y=1, x=1, xs=None, w=1, s=1, bias=None, M=2, N=64, K=64, xt=L.DT_BFLOAT16, yt=L.DT_BFLOAT16,
             ws=16, need=1 << 20, gate=None, up=None, w2=1, s2=1)
    a.update(kw)
    p = lambda k: P(a[k])
    tail = (a["M"], a["N"], a["K"], a["xt"], a["yt"], p("ws"), a["need"], None)
    if fn == "mi_int8_matmul":
        return L.lib().mi_int8_matmul(p("y"), p("x"), p("xs"), p("w"), p("s"), p("bias"), *tail)
    return L.lib().mi_int8_gate_up_swiglu(p("y"), p("gate"), p("up"), p("x"), p("xs"), p("w"), p("s"), p("w2"),
                                          p("s2"), *tail)


BAD = [(dict(M=-1), L.MI_ERR_INVALID, "negative"), (dict(K=0), L.MI_ERR_INVALID, "K must"),
       (dict(N=1 << 31), L.MI_ERR_INVALID, "too large"), (dict(K=131072), L.MI_ERR_UNSUPPORTED, "131071"),
       (dict(xt=L.DT_UINT8), L.MI_ERR_UNSUPPORTED, "x dtype"), (dict(yt=L.DT_INT8), L.MI_ERR_UNSUPPORTED, "y dtype"),
       (dict(xs=1), L.MI_ERR_INVALID, "x_scales"), (dict(xt=L.DT_INT8), L.MI_ERR_INVALID, "null"),
       (dict(y=None), L.MI_ERR_INVALID, "null"), (dict(w=None), L.MI_ERR_INVALID, "null"),
       (dict(ws=None), L.MI_ERR_WORKSPACE, "workspace"), (dict(need=8), L.MI_ERR_WORKSPACE, "workspace"),
       (dict(ws=8), L.MI_ERR_INVALID, "aligned"), (dict(M=1 << 29, N=1 << 20), L.MI_ERR_UNSUPPORTED, "too large")]


@pytest.mark.parametrize("fn", ["mi_int8_matmul", "mi_int8_gate_up_swiglu"])
@pytest.mark.parametrize("kw,code,msg", BAD)
def test_forward_refusals(fn, kw, code, msg):
    kw = dict(dict(M=40), **kw)
    assert _forward(fn, **kw) == code
    assert msg in L.last_error()


def test_gate_up_refusals():
    fn = "mi_int8_gate_up_swiglu"
    assert _forward(fn, gate=1) == L.MI_ERR_INVALID and "together" in L.last_error()
    assert _forward(fn, w2=None) == L.MI_ERR_INVALID
    assert _forward(fn, s2=None) == L.MI_ERR_INVALID
    assert _forward(fn, M=0, w2=None) == L.MI_OK


def test_empty_outputs_are_no_ops():
    assert _forward(M=0, y=None, x=None, ws=None) == L.MI_OK
    assert _forward(N=0, y=None, w=None, s=None, ws=None) == L.MI_OK
    lib = L.lib()
    assert lib.mi_int8_quantize(None, None, None, 0, 64, L.DT_BFLOAT16, None) == L.MI_OK
    assert lib.mi_int8_matmul_backward(None, None, None, None, 0, 8, 8, L.DT_BFLOAT16, None, 0, None) == L.MI_OK
    assert lib.mi_int8_matmul_backward(None, None, None, None, 8, 8, 0, L.DT_BFLOAT16, None, 0, None) == L.MI_OK


def test_quantize_refusals():
    f = L.lib().mi_int8_quantize
    assert f(P(1), P(1), P(1), -1, 8, L.DT_BFLOAT16, None) == L.MI_ERR_INVALID
    assert f(P(1), P(1), P(1), 1, 0, L.DT_BFLOAT16, None) == L.MI_ERR_INVALID
    assert f(P(1), P(1), P(1), 1, 8, L.DT_INT8, None) == L.MI_ERR_UNSUPPORTED
    assert f(None, P(1), P(1), 1, 8, L.DT_BFLOAT16, None) == L.MI_ERR_INVALID


@pytest.mark.parametrize("kw,code", [(dict(M=-1), L.MI_ERR_INVALID), (dict(N=0), L.MI_ERR_INVALID),
                                     (dict(t=L.DT_INT8), L.MI_ERR_UNSUPPORTED), (dict(dy=None), L.MI_ERR_INVALID),
                                     (dict(gate=None), L.MI_ERR_INVALID), (dict(dgate=None), L.MI_ERR_INVALID),
                                     (dict(ws=None), L.MI_ERR_WORKSPACE), (dict(need=64), L.MI_ERR_WORKSPACE),
                                     (dict(ws=4), L.MI_ERR_INVALID), (dict(K=1 << 31), L.MI_ERR_INVALID),
                                     (dict(M=1 << 29, K=1 << 20), L.MI_ERR_UNSUPPORTED),
                                     (dict(M=1 << 28, N=1 << 28, K=1), L.MI_ERR_UNSUPPORTED)])
def test_backward_refusals(kw, code):
    a = dict(dx=1, dgate=1, dup=1, dy=1, gate=1, up=1, w=1, s=1, M=40, N=64, K=64, t=L.DT_BFLOAT16, ws=16,
             need=1 << 20)
    a.update(kw)
    p = lambda k: P(a[k])
    rc = L.lib().mi_int8_gate_up_swiglu_backward(p("dx"), p("dgate"), p("dup"), p("dy"), p("gate"), p("up"), p("w"),
                                                 p("s"), p("w"), p("s"), a["M"], a["N"], a["K"], a["t"], p("ws"),
                                                 a["need"], None)
    assert rc == code, L.last_error()
    if "gate" not in kw and "dgate" not in kw:
        rc = L.lib().mi_int8_matmul_backward(p("dx"), p("dy"), p("w"), p("s"), a["M"], a["N"], a["K"], a["t"],
                                             p("ws"), a["need"], None)
        assert rc == code, L.last_error()


def test_workspace_sizes():
    lib = L.lib()
    assert lib.mi_int8_forward_workspace(64, 64, 64, 1, L.DT_INT8) >= 0
    assert lib.mi_int8_forward_workspace(-1, 64, 64, 1, L.DT_INT8) == -1
    assert lib.mi_int8_forward_workspace(1, 64, 64, 3, L.DT_INT8) == -1
    assert lib.mi_int8_backward_workspace(1, 64, 64, 1, L.DT_INT8) == -1
    assert lib.mi_int8_backward_workspace(1 << 28, 1 << 28, 64, 1, L.DT_BFLOAT16) == -1
    one, two = (lib.mi_int8_backward_workspace(64, 64, 64, b, L.DT_BFLOAT16) for b in (1, 2))
    assert two > one > 0


def test_python_refuses_host_tensors():
    x, w, s = torch.zeros(2, 8, dtype=torch.bfloat16), torch.zeros(4, 8, dtype=torch.int8), torch.ones(4)
    for call in (lambda: mi_qmm.int8_quantize(x), lambda: mi_qmm.int8_matmul(x, w, s),
                 lambda: mi_qmm.int8_gate_up_swiglu(x, w, s, w, s), lambda: mi_qmm.int8_matmul_backward(x, w, s),
                 lambda: mi_qmm.int8_gate_up_swiglu_backward(x, x, x, w, s, w, s)):
        with pytest.raises(mi_qmm.MiError):
            call()


def test_reference_formulas():
    """The reference itself: codes by brute force, gradients against differences."""
    x = torch.tensor([[127.0, 0.5, 1.5, -2.5, 126.5], [254.0, 1.0, 3.0, -5.0, 253.0], [0.0] * 5])
    q, s = R.quantize(x)
    assert s.tolist() == [1.0, 2.0, 0.0]
    assert q.tolist() == [[127, 0, 2, -2, 126], [127, 0, 2, -2, 126], [0] * 5]
    g = torch.Generator().manual_seed(1)
    dy, a, b = (torch.randn(3, 4, generator=g, dtype=torch.float64) for _ in range(3))
    f = lambda a, b: (a * torch.special.expit(a) * b * dy)
    da, db, _, _ = R.grads(dy, a, b)
    e = 1e-6
    assert torch.allclose(da, (f(a + e, b) - f(a - e, b)) / (2 * e), atol=1e-8)
    assert torch.allclose(db, (f(a, b + e) - f(a, b - e)) / (2 * e), atol=1e-8)
