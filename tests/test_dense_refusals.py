"""CPU: what the dense operators on device tensors refuse, in Python before anything reaches the GPU and at the C entry."""
import ctypes as C

import pytest

torch = pytest.importorskip("torch")

from sclens_amd import _lib, dense  # noqa: E402

BF16, F32 = torch.bfloat16, torch.float32


def t(*shape, dtype=F32):
    return torch.zeros(*shape, dtype=dtype)


class _Gpu(torch.Tensor):
    """a CPU tensor that says it is on a GPU: the checks of shapes and strides run, nothing may go further"""

    @property
    def device(self):
        return torch.device("cuda", 0)

    @property
    def is_cuda(self):
        return True

    def get_device(self):
        return 0


def g(*shape, dtype=F32):
    return torch.zeros(*shape, dtype=dtype).as_subclass(_Gpu)


@pytest.fixture(autouse=True)
def no_call(monkeypatch):
    def stop(*a, **k):
        raise AssertionError("a call that has to be refused went on to the library")

    monkeypatch.setattr(dense, "_context", stop)


@pytest.mark.parametrize("call,kind,text", [
    (lambda: dense.linear([[1.0]], t(1, 1)), TypeError, "torch tensor"),
    (lambda: dense.linear(t(2, 3), t(4, 3)), ValueError, "GPU"),
    (lambda: dense.linear(t(2, 3, dtype=torch.float64), t(4, 3)), TypeError, "float64"),
    (lambda: dense.linear(t(2, 3).requires_grad_(True), t(4, 3)), ValueError, "gradient"),
    (lambda: dense.linear(g(2, 3), g(4, 3), activation="tanh"), ValueError, "unknown activation"),
    (lambda: dense.linear(g(2, 3), g(4, 5)), ValueError, "expected"),
    (lambda: dense.linear(g(2, 3), g(3)), ValueError, "expected"),
    (lambda: dense.linear(g(2, 3), g(4, 3, dtype=BF16)), ValueError, "weight"),
    (lambda: dense.linear(g(2, 3), t(4, 3)), ValueError, "weight"),
    (lambda: dense.linear(g(2, 3), g(4, 3), bias=g(3)), ValueError, "bias"),
    (lambda: dense.linear(g(2, 3), g(4, 3), bias=g(8)[::2]), ValueError, "contiguous"),
    (lambda: dense.linear(g(2, 3), g(4, 3), residual=g(4)), ValueError, "residual"),
    (lambda: dense.linear(g(2, 3), g(4, 3), residual=g(1, 4).expand(2, 4)), ValueError, "overlap"),
    (lambda: dense.linear(g(3, 2).t(), g(4, 3)), ValueError, "rows have to be contiguous"),
    (lambda: dense.linear(g(2, 3), g(3, 4).t()), ValueError, "rows have to be contiguous"),
    (lambda: dense.linear(g(5, 2, 3).transpose(0, 1), g(4, 3)), ValueError, "leading axes"),
    (lambda: dense.linear_backward(g(2, 4), g(2, 3), g(4, 3), activation="silu"), ValueError, "preact"),
    (lambda: dense.linear_backward(g(2, 4), g(2, 3), g(4, 3), preact=g(2, 5), activation="silu"), ValueError, "preact"),
    (lambda: dense.linear_backward(g(2, 4), None, g(4, 3)), ValueError, "dweight needs x"),
    (lambda: dense.linear_backward(g(2, 4), g(2, 3), None), ValueError, "dx needs weight"),
    (lambda: dense.linear_backward(g(2, 4), g(3, 3), g(4, 3)), ValueError, "x: shape"),
    (lambda: dense.linear_backward(g(2, 4), g(2, 3), g(4, 2)), ValueError, "weight: shape"),
    (lambda: dense.linear_backward(g(4, 2).t(), g(2, 3), g(4, 3)), ValueError, "rows have to be contiguous"),
    (lambda: dense.orthogonalize(g(5)), ValueError, "expected"),
    (lambda: dense.orthogonalize(t(5, 5)), ValueError, "GPU"),
    (lambda: dense.orthogonalize(g(5, 5), steps=0), ValueError, "step"),
    (lambda: dense.orthogonalize(g(5, 5), coefficients=[]), ValueError, "coefficients"),
    (lambda: dense.orthogonalize(g(5, 5), coefficients=[(1.0, 2.0)]), ValueError, "coefficients"),
    (lambda: dense.orthogonalize(g(5, 6).t()), ValueError, "rows have to be contiguous"),
    (lambda: dense.orthogonalize(g(2, 3, 4, 5).transpose(0, 1)), ValueError, "leading axes"),
])
def test_refused_before_the_library(call, kind, text):
    with pytest.raises(kind, match=text):
        call()


def test_c_entries_without_a_context():
    lib = _lib.load()
    n = C.c_int64(0)
    assert lib.sclens_hip_linear(None, None, 0, 1, 1, 1, None, 1, None, 1, None, None, 1, 0, None, 1, None, 1, None, C.byref(n)) == 1
    assert lib.sclens_hip_linear_backward(None, None, 0, 1, 1, 1, None, 1, None, 1, None, 1, None, 1, 0, None, 1, None, 1, None, None,
                                          C.byref(n)) == 1
    assert lib.sclens_hip_orthogonalize(None, None, 0, 1, 1, 1, None, 1, 1, None, 1, 1, 1, None, 0.0, None, C.byref(n)) == 1


def test_library_loaded_before_torch_is_refused(monkeypatch):
    monkeypatch.undo()
    monkeypatch.setattr(_lib, "shares_torch_runtime", False)

    class Ctx:
        device = 0

    with pytest.raises(RuntimeError, match="import torch"):
        dense._context(0, Ctx())
    with pytest.raises(ValueError, match="context on device"):
        dense._context(1, Ctx())


def test_forward_mode_tangents_are_refused():
    """a dual tensor does not require a gradient: its tangent would be dropped in silence"""
    from torch.autograd import forward_ad

    calls = [
        (lambda d: dense.linear(d(2, 3), g(4, 3)), "x carries"),
        (lambda d: dense.linear(g(2, 3), d(4, 3)), "weight carries"),
        (lambda d: dense.linear(g(2, 3), g(4, 3), bias=d(4)), "bias carries"),
        (lambda d: dense.linear(g(2, 3), g(4, 3), residual=d(2, 4)), "residual carries"),
        (lambda d: dense.linear_backward(d(2, 4), g(2, 3), g(4, 3)), "grad carries"),
        (lambda d: dense.linear_backward(g(2, 4), d(2, 3), g(4, 3)), "x carries"),
        (lambda d: dense.linear_backward(g(2, 4), g(2, 3), d(4, 3)), "weight carries"),
        (lambda d: dense.linear_backward(g(2, 4), g(2, 3), g(4, 3), preact=d(2, 4), activation="silu"), "preact carries"),
        (lambda d: dense.orthogonalize(d(5, 6)), "x carries"),
    ]
    with forward_ad.dual_level():
        def dual(*shape):
            v = forward_ad.make_dual(g(*shape), torch.ones(shape))
            assert v.is_cuda and not v.requires_grad
            return v

        for call, text in calls:
            with pytest.raises(ValueError, match=text):
                call(dual)
            with torch.no_grad(), pytest.raises(ValueError, match=text):  # no_grad does not switch tangents off
                call(dual)
