"""Host-side checks of the 4-bit weights' and the experts' entry points: bad
sizes, types and pointers are refused before any launch (no GPU needed), and the
64-bit restatements the GPU tests compare with agree with themselves."""

from __future__ import annotations

import ctypes

import pytest
import torch

import ffn_oracle as fo

P = ctypes.c_void_p(64)          # 16-byte aligned, never read
ODD = ctypes.c_void_p(68)


def linear(qm, act=1, m=1, n=16, k=64, codes=P, scales=P, x=P, ldx=64, rows=(16,), outs=(64,)):
    seg = (ctypes.c_int * len(rows))(*rows)
    out = (ctypes.c_void_p * len(outs))(*outs)
    return qm.native.load().qm_mx4_linear(act, m, n, k, codes, scales, x, ldx, len(rows), seg, out, None)


@pytest.mark.parametrize("kw,code", [
    (dict(act=7), -2), (dict(m=0), -1), (dict(n=0), -1), (dict(k=48, ldx=48), -1), (dict(k=0), -1), (dict(codes=None), -1),
    (dict(scales=None), -1), (dict(x=None), -1), (dict(x=ODD), -1), (dict(codes=ODD), -1), (dict(ldx=63), -1),
    (dict(ldx=68), -1), (dict(rows=(8, 9), outs=(64, 64)), -1), (dict(rows=(16, 0), outs=(64, 64)), -1),
    (dict(outs=(None,)), -1), (dict(n=9, rows=(1,) * 9, outs=(64,) * 9), -1), (dict(m=16 * 65535 + 1), -1)])
def test_mx4_linear_refuses(qm, kw, code):
    assert linear(qm, **kw) == code
    assert b"qm_mx4_linear" in qm.native.load().qm_last_error()


def test_mx4_conversions_refuse(qm):
    lib = qm.native.load()
    assert lib.qm_mx4_quantize(7, 1, 16, 64, P, P, P, None) == -2
    assert lib.qm_mx4_quantize(1, 1, 16, 40, P, P, P, None) == -1
    assert lib.qm_mx4_quantize(1, 0, 16, 64, P, P, P, None) == -1
    assert lib.qm_mx4_quantize(1, 1, 16, 64, ODD, P, P, None) == -1
    assert lib.qm_mx4_quantize(1, 1, 16, 64, P, P, None, None) == -1
    assert lib.qm_mx4_dequantize(7, 1, 16, 64, P, P, P, None) == -2
    assert lib.qm_mx4_dequantize(1, 1, 16, 64, P, P, ODD, None) == -1
    assert lib.qm_mx4_layout(1, 1, 16, 33, P, P, P, P, None) == -1
    assert lib.qm_mx4_layout(1, 1, 16, 64, P, P, ODD, P, None) == -1
    assert lib.qm_mx4_layout(0, 1 << 24, 1 << 20, 1 << 12, P, P, P, P, None) == -5      # too many tiles
    assert lib.qm_tile_weight(7, 1, 16, 64, P, P, None) == -2
    assert lib.qm_tile_weight(1, 1, 16, 65, P, P, None) == -1
    assert lib.qm_tile_weight(1, 1, 16, 64, P, None, None) == -1
    assert lib.qm_mx4_code_bytes(1, 16, 40) == 0
    assert lib.qm_mx4_code_bytes(3, 17, 160) == 3 * 2 * 2 * 1024


def test_moe_route_refuses(qm):
    lib = qm.native.load()

    def route(act=1, rows=2, hidden=64, experts=8, top_k=2, x=P, ldx=64, router=P, ids=P, weights=P, ws=P, nbytes=1 << 20):
        return lib.qm_moe_route(act, rows, hidden, experts, top_k, 1, x, ldx, router, ids, weights, ws, nbytes, None)

    assert route(act=3) == -2
    assert route(rows=0) == -1 and route(rows=262141) == -1
    assert route(hidden=40, ldx=40) == -1 and route(hidden=0) == -1
    assert route(experts=0, top_k=0) == -5 and route(experts=1025) == -5
    assert route(top_k=0) == -1 and route(top_k=9) == -1 and route(experts=64, top_k=33) == -1
    assert route(ldx=32) == -1 and route(ldx=68) == -1
    assert route(x=None) == -1 and route(ws=None) == -1 and route(x=ODD) == -1 and route(router=ODD) == -1
    assert route(nbytes=lib.qm_moe_route_workspace(2, 8) - 1) == -4
    assert b"qm_moe_route" in lib.qm_last_error()
    assert lib.qm_moe_route_workspace(2, 8) >= 2 * 8 * 8
    assert lib.qm_moe_route_workspace(0, 8) == 0 and lib.qm_moe_route_workspace(2, 1025) == 0


def test_moe_refuses(qm):
    n = qm.native
    lib = n.load()

    def run(x=P, ldx=64, out=P, ws=P, nbytes=1 << 30, weights=None, **geom):
        g = dict(rows=2, hidden=64, inter=32, experts=8, shared=1, top_k=2, normalize=1, act_dtype=1, weight_format=0)
        g.update(geom)
        w = n.MoeWeightPtrs(*([64] * 14))
        for name, v in (weights or {}).items():
            setattr(w, name, v)
        return lib.qm_moe(ctypes.byref(n.MoeGeom(**g)), ctypes.byref(w), x, ldx, out, ws, nbytes, None)

    assert run(act_dtype=2) == -2 and run(weight_format=2) == -2
    assert run(rows=0) == -1 and run(hidden=33) == -1 and run(inter=0) == -1 and run(inter=40) == -1
    assert run(experts=2000) == -5 and run(top_k=9) == -1 and run(shared=-1) == -1 and run(shared=33) == -1
    assert run(ldx=32) == -1 and run(x=None) == -1 and run(out=None) == -1 and run(out=ODD) == -1 and run(ws=None) == -1
    assert run(weights={"gate": None}) == -1 and run(weights={"down": 72}) == -1
    assert run(weights={"shared_up": None}) == -1 and run(weights={"shared_router": 72}) == -1
    assert run(weight_format=1, weights={"up_scales": None}) == -1
    assert run(weight_format=1, weights={"shared_down_scales": None}) == -1
    assert run(nbytes=256) == -4
    assert b"qm_moe" in lib.qm_last_error()
    assert lib.qm_moe(None, None, P, 64, P, P, 1 << 30, None) == -1
    assert lib.qm_moe_workspace(None) == 0


def test_python_refuses_host_tensors(qm):
    x = torch.zeros(2, 64)
    for call in (lambda: qm.mx4_quantize(x), lambda: qm.moe_route(x, x, 1), lambda: qm.mx4_linear(x, None),
                 lambda: qm.MoeWeights(x, x, x, x, 1)):
        with pytest.raises(ValueError, match="GPU"):
            call()
    with pytest.raises(ValueError, match="uint8"):
        qm.Mx4Weight.from_codes(x, x)


def test_oracle_quantisation_is_nearest_and_round_trips():
    g = torch.Generator().manual_seed(1)
    w = torch.randn(6, 96, generator=g) * torch.logspace(-8, 8, 6)[:, None]
    codes, scales = fo.mx4_encode(w)
    v = fo.mx4_decode(codes, scales)
    # re-quantising the values gives them back, unless their largest fell to the scale below
    again = fo.mx4_decode(*fo.mx4_encode(v.float()))
    assert torch.equal(again, v)
    # no other code of the block is nearer
    grid = torch.tensor(fo.GRID + [-x for x in fo.GRID], dtype=torch.float64)
    s = torch.pow(2.0, scales.double() - 127).repeat_interleave(32, -1)
    best = (w.double()[..., None] - grid * s[..., None]).abs().min(-1).values
    assert torch.equal((w.double() - v).abs(), best)
    assert torch.equal(fo.mx4_decode(torch.tensor([[0x21] * 16], dtype=torch.uint8), torch.tensor([[128]], dtype=torch.uint8)),
                       torch.tensor([[1.0, 2.0] * 16], dtype=torch.float64))
