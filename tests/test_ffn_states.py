"""Host-side checks of the experts' and the 4-bit weights' Python layer that need no
GPU: what it refuses before any tensor is read."""

from __future__ import annotations

import pytest
import torch
import torch.autograd.forward_ad as fw
from torch.fx.experimental.proxy_tensor import make_fx


def test_tangents_are_refused(qm):
    x = torch.zeros(2, 64)
    with fw.dual_level():
        d = fw.make_dual(x, torch.ones_like(x))
        for call in (lambda: qm.mx4_quantize(d), lambda: qm.mx4_linear(d, None), lambda: qm.moe_route(d, x, 1),
                     lambda: qm.moe(d[:1], None), lambda: qm.MoeWeights(d, x, x, x, 1)):
            with pytest.raises(RuntimeError, match="tangent"):
                call()
            with torch.no_grad(), pytest.raises(RuntimeError, match="tangent"):
                call()
        with pytest.raises(ValueError, match="GPU"):                # without a tangent: as ever
            qm.mx4_quantize(x)


def test_recording_is_refused(qm):
    """The one place that every launch passes."""
    from importlib import import_module
    mx4 = import_module(qm.__name__ + ".mx4")

    def f(x):
        mx4.refuse_recording()
        return x + 1

    x = torch.zeros(2)
    f(x)
    with pytest.raises(RuntimeError, match="traced"):
        torch.jit.trace(f, x)
    with pytest.raises(RuntimeError, match="traced"):
        make_fx(f)(x)
    # a launch without a device: refused before that is looked at
    with pytest.raises(RuntimeError, match="traced"):
        torch.jit.trace(lambda v: (mx4.launch("qm_mx4_quantize", None), v + 1)[1], x)
    f(x)
