"""Host-side checks of the experts' and the 4-bit weights' entry points that need no
GPU: what they refuse before any tensor is read."""

from __future__ import annotations

import copy
import ctypes
import pickle

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


@pytest.mark.parametrize("off", [1, 2, 3])
@pytest.mark.parametrize("m", [1, 200])
def test_scales_that_are_not_whole_words_are_refused(qm, m, off):
    """For the few-row kernels, which read bytes, as for the staged ones, which read
    words."""
    n = qm.native
    lib = n.load()
    p = ctypes.c_void_p(64)
    seg, out = (ctypes.c_int * 1)(4096), (ctypes.c_void_p * 1)(64)
    assert lib.qm_mx4_linear(1, m, 4096, 64, p, ctypes.c_void_p(64 + off), p, 64, 1, seg, out, None) == -1
    assert b"scales" in lib.qm_last_error()
    g = n.MoeGeom(m, 64, 32, 8, 1, 2, 1, 1, n.QM_W_MX4)
    for name in ("gate", "up", "down", "shared_gate", "shared_up", "shared_down"):
        w = n.MoeWeightPtrs(*([64] * 14))
        setattr(w, name + "_scales", 64 + off)
        assert lib.qm_moe(ctypes.byref(g), ctypes.byref(w), p, 64, p, p, 1 << 30, None) == -1, name
        assert b"scales" in lib.qm_last_error()


def test_a_4_bit_weight_is_as_large_as_its_shape(qm):
    """Tiles that a kernel would read past are refused where the weight is made."""
    tiles = lambda n: torch.zeros(n * 1088, dtype=torch.uint8)  # noqa: E731
    assert qm.Mx4Weight(tiles(4), (17, 160)).code_bytes == 4 * 1024
    assert qm.Mx4Weight(tiles(12), (3, 17, 160)).mats == 3
    for data, shape in ((tiles(3), (17, 160)), (tiles(5), (17, 160)), (tiles(4), (3, 17, 160)), (tiles(4).int(), (17, 160)),
                        (tiles(8)[::2], (17, 160)), (torch.zeros(4 * 1088 + 1, dtype=torch.uint8)[1:], (17, 160))):
        with pytest.raises(ValueError, match="tiles of"):
            qm.Mx4Weight(data, shape)
    with pytest.raises(ValueError, match="multiple of 32"):
        qm.Mx4Weight(tiles(4), (17, 150))


def test_weights_do_not_change_once_made(qm):
    """Calls keep their addresses and sizes."""
    q = qm.Mx4Weight(torch.zeros(4 * 1088, dtype=torch.uint8), (17, 160))
    w = qm.MoeWeights.__new__(qm.MoeWeights)
    w.top_k = 2
    for obj, name, value in ((q, "data", torch.zeros(1088, dtype=torch.uint8)), (q, "shape", (16, 32)), (q, "code_bytes", 1),
                             (w, "top_k", 3)):
        with pytest.raises(AttributeError, match="does not change"):
            setattr(obj, name, value)
        with pytest.raises(AttributeError, match="does not change"):
            delattr(obj, name)
    assert q.data.numel() == 4 * 1088 and w.top_k == 2
    for other in (copy.copy(q), copy.deepcopy(q), pickle.loads(pickle.dumps(q))):
        assert other.shape == q.shape and torch.equal(other.data, q.data)


def test_the_experts_fields_stand_behind_the_configurations_others(qm):
    """Configurations made by position keep their meaning."""
    c = qm.MixConfig(1024, 1e-5, 8, 1, 128, 1e6, 32, [6, 5, 5], 2, 2, 64, 512, 32, 16, 8, 64, 3, "sigmoid", 2, 160, 128)
    assert (c.hc_count, c.hc_lowrank, c.page_size) == (2, 160, 128)
    assert (c.num_experts_per_tok, c.norm_topk_prob, c.shared_expert) == (8, True, True)
