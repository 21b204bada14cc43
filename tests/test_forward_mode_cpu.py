"""The routing, sort and microscaled operators have no forward-mode derivatives: a tensor that carries a tangent is refused, where its
values alone would give a result without one. Nothing here needs a GPU: the refusal comes before the launch."""
import pytest
import torch
import torch.autograd.forward_ad as fw

import flux_b200 as flux
from flux_b200 import _lib, moe, mx


class _Library:
    """Takes every call."""

    def __getattr__(self, name):
        return lambda *_: _lib.FLUXB_OK


@pytest.fixture(autouse=True)
def no_gpu(monkeypatch):
    for module in (moe, mx):
        monkeypatch.setattr(module, "_on_device", lambda t: True)
        monkeypatch.setattr(module, "_cur_stream", lambda: None)
    monkeypatch.setattr(mx, "_cur_device", lambda: -1)
    monkeypatch.setattr(mx, "_comm", lambda: type("", (), {"handle": None}))
    monkeypatch.setattr(_lib, "load", _Library)


INDEX = torch.zeros(4, 2, dtype=torch.int32)
SPLITS = torch.zeros(3, dtype=torch.int32)


def _matrix(rows):
    return mx.MXTensor._of(torch.zeros(rows, 16, dtype=torch.uint8), torch.zeros(1, 1, 512, dtype=torch.uint8))


CALLS = {
    "moe_route": ((4, 8), lambda t: flux.moe_route(t, 2)),
    "moe_permute": ((4, 8), lambda t: flux.moe_permute(t, SPLITS, INDEX)),
    "moe_unpermute rows": ((8, 8), lambda t: flux.moe_unpermute(t, SPLITS, INDEX)),
    "moe_unpermute weights": ((4, 2), lambda t: flux.moe_unpermute(torch.zeros(8, 8), SPLITS, INDEX, t)),
    "mx_quantize": ((4, 32), lambda t: flux.mx_quantize(t)),
    "mx_gemm": ((5,), lambda t: flux.mx_gemm(_matrix(4), _matrix(5), bias=t, output_dtype=torch.float32)),
}


@pytest.mark.parametrize("grad", [True, False])
@pytest.mark.parametrize("name", CALLS)
def test_a_tangent_is_refused(name, grad):
    shape, call = CALLS[name]
    with fw.dual_level(), torch.set_grad_enabled(grad):
        call(torch.zeros(shape))  # without a tangent it is an ordinary call
        with pytest.raises(RuntimeError, match=f"{name.split()[0]} has no forward-mode derivative"):
            call(fw.make_dual(torch.zeros(shape), torch.ones(shape)))
        with pytest.raises(RuntimeError, match=f"{name.split()[0]}.* has no (forward-mode|gradient)"):
            call(fw.make_dual(torch.zeros(shape, requires_grad=True), torch.ones(shape)))


@pytest.mark.parametrize("name", ["moe_route", "moe_permute", "moe_unpermute rows", "moe_unpermute weights"])
def test_a_tangent_of_a_gradient_is_refused(name):
    shape, call = CALLS[name]
    x = torch.zeros(shape, requires_grad=True)
    out = call(x)
    out = out[1] if name == "moe_route" else out
    with fw.dual_level():
        torch.autograd.grad(out, x, torch.ones_like(out), retain_graph=True)
        with pytest.raises(RuntimeError, match=f"{name.split()[0]}.* has no forward-mode derivative"):
            torch.autograd.grad(out, x, fw.make_dual(torch.ones_like(out), torch.ones_like(out)))
