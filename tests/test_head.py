"""The output-head entry points without a GPU: argument checks that need no
device, and the 64-bit results the GPU tests compare with, against
independent forms."""
import ctypes

import pytest
import torch

import head_cases as H
from qwenium_b200 import build as qbuild
from qwenium_b200 import qsamp


@pytest.fixture(scope="module")
def lib():
    qbuild.build()
    return qsamp.load()


def test_entry_points_refuse_no_context(lib):
    head = qsamp._Head()
    prod = qsamp._Fp8Product()
    assert lib.qsamp_head_workspace(None, 1, 1, 8, 0) == -1
    assert lib.qsamp_head_loss(None, ctypes.byref(head), None, None, None, 0, None) == 1
    assert lib.qsamp_head_loss_grad(None, ctypes.byref(head), None, None, None, 0, None, 0, None, 0, None) == 1
    assert lib.qsamp_quantize_fp8(None, None, 0, 1, 1, 1, 1, None, 1, None, 1, None) == 1
    assert lib.qsamp_matmul_fp8(None, ctypes.byref(prod), None) == 1


def test_tensor_checks():
    """Every tensor argument is checked before a pointer leaves Python."""
    ctx = object.__new__(qsamp.Context)
    ctx.device = 0
    x = torch.zeros((4, 8))
    with pytest.raises(qsamp.QsampError, match="x: expected a tensor on cuda:0, got cpu") as e:
        ctx._tensor("x", x, (torch.float32,), (None, None))
    assert e.value.status == 1

    class OnCuda:
        device = torch.device("cuda", 0)
        is_cuda = True

        def get_device(self):
            return 0

        def __init__(self, t):
            self.t = t

        def __getattr__(self, k):
            return getattr(self.t, k)

    with pytest.raises(qsamp.QsampError, match="expected torch.bfloat16, got torch.float32"):
        ctx._tensor("x", OnCuda(x), (torch.bfloat16,), (None, None))
    with pytest.raises(qsamp.QsampError, match="expected shape"):
        ctx._tensor("x", OnCuda(x), (torch.float32,), (None, 9))
    with pytest.raises(qsamp.QsampError, match="expected shape"):
        ctx._tensor("x", OnCuda(x), (torch.float32,), (4,))
    with pytest.raises(qsamp.QsampError, match="unit stride"):
        ctx._tensor("x", OnCuda(x.t()), (torch.float32,), (8, 4))
    ctx._tensor("x", OnCuda(x), (torch.float32,), (4, 8))


@pytest.mark.parametrize("cap", [0.0, 5.0])
def test_exact_gradients_are_the_derivatives(cap):
    h, w, t, g = H.head_inputs(9, 50, 16, seed=1)
    want = H.head_exact(h, w, t, g, cap)
    hd, wd = h.double().requires_grad_(), w.double().requires_grad_()
    z = hd @ wd.t()
    if cap:
        z = cap * torch.tanh(z / cap)
    live = t >= 0
    loss = torch.nn.functional.cross_entropy(z, t.long().clamp(min=0), reduction="none")
    loss = torch.where(live, loss, 0.0)
    (loss * g.double()).sum().backward()
    torch.testing.assert_close(want["loss"], loss.detach(), rtol=1e-12, atol=1e-12)
    torch.testing.assert_close(want["dh"], hd.grad, rtol=1e-11, atol=1e-12)
    torch.testing.assert_close(want["dw"], wd.grad, rtol=1e-11, atol=1e-12)


def test_exact_quantiser_is_the_formats_rounding():
    """With a scale of 1 the values are torch's own rounding to e4m3 (saturated)."""
    g = torch.Generator().manual_seed(3)
    x = (torch.randn((6, 256), generator=g) * 60).clamp(-448, 448)
    x[:, 0] = 448.0
    x[:, 128] = -448.0
    q, s = H.quant_exact(x, 1)
    assert (s == 1).all()
    assert torch.equal(q, x.to(torch.float8_e4m3fn).double())
