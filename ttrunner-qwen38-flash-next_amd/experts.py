"""The mixture-of-experts layer: routing and the chosen experts' gated FFN.

``moe_route`` picks each token's experts, ``moe`` is the whole layer over a
``MoeWeights`` (reference/model.py:387-417): router, the chosen experts, and the
shared experts that every token takes. ``Qwen4MixModel._moe`` builds the weights
of a layer from the model's store, ``MixDecoder(ffn=True)`` runs it inside a
decode step.

Everything runs in the HIP kernels of libqwen4mix.so on the current stream of
the tensors' device. Nothing here is differentiable.
"""

from __future__ import annotations

import ctypes
import functools

import torch

from . import native
from .mx4 import BLOCK, Mx4Weight, SetOnce, activation_rows, check_input, dense, launch

MAX_EXPERTS, MAX_TOP_K, MAX_SHARED = 1024, 32, 32


@functools.lru_cache(256)
def _route_bytes(rows: int, experts: int) -> int:
    return native.load().qm_moe_route_workspace(rows, experts)


def _check_router(x: torch.Tensor, router: torch.Tensor, top_k: int) -> None:
    experts, hidden = router.shape
    if x.dim() == 0 or x.shape[-1] != hidden:
        raise ValueError(f"x must be [..., {hidden}], got {tuple(x.shape)}")
    if x.dtype != router.dtype or x.device != router.device:
        raise ValueError(f"x is {x.dtype} on {x.device}, the router {router.dtype} on {router.device}")
    if not 1 <= top_k <= min(experts, MAX_TOP_K):
        raise ValueError(f"top_k must be 1 to {min(experts, MAX_TOP_K)}, got {top_k}")


def _check_router_shape(router: torch.Tensor) -> None:
    check_input(router, "the router")
    if router.dim() != 2 or not 1 <= router.shape[0] <= MAX_EXPERTS:
        raise ValueError(f"the router must be [experts, hidden] with 1 to {MAX_EXPERTS} experts, got "
                         f"{tuple(router.shape)}")
    if router.shape[1] == 0 or router.shape[1] % BLOCK:
        raise ValueError(f"hidden must be a multiple of {BLOCK}, got {router.shape[1]}")


def moe_route(x: torch.Tensor, router: torch.Tensor, top_k: int, normalize: bool = True):
    """The experts of each token: x [..., hidden], router [experts, hidden] (one
    type, float32 or bfloat16) -> (ids int32 [..., top_k], weights float32
    [..., top_k]).

    ids are the experts of the largest logits x router^T in falling order (equal
    ones: the lower index first; NaN above every number), weights their softmax
    over all experts, or over the chosen ones when ``normalize``. The order is that of
    sums in float64, so a token's experts do not depend on the rows beside it. Its
    weights do by their last bits: with many rows they come of logits summed in
    float, 128 products at a time (include/qwen4mix.h gives the bound)."""
    act = check_input(x, "x")
    _check_router_shape(router)
    _check_router(x, router, top_k)
    experts, hidden = router.shape
    shape, device = x.shape[:-1] + (top_k,), x.device
    ids = torch.empty(shape, dtype=torch.int32, device=device)
    weights = torch.empty(shape, dtype=torch.float32, device=device)
    m = x.numel() // hidden
    if m:
        xr, ldx = activation_rows(x)
        rc = dense(router)
        nbytes = _route_bytes(m, experts)
        ws = torch.empty(nbytes, dtype=torch.uint8, device=device)
        launch("qm_moe_route", device, act, m, hidden, experts, top_k, 1 if normalize else 0, xr.data_ptr(), ldx,
               rc.data_ptr(), ids.data_ptr(), weights.data_ptr(), ws.data_ptr(), nbytes)
    return ids, weights


def _copy(t: torch.Tensor) -> torch.Tensor:
    """t in memory of its own, as the other weights have it: a loader may read the
    next layer into the same buffer."""
    return t.detach().clone(memory_format=torch.contiguous_format)


class _Tiles(SetOnce):
    """A weight [mats, n, k] of the activations' type in the kernels' tile order."""

    def __init__(self, w: torch.Tensor):
        mats, n, k = w.shape
        self.shape = w.shape
        wc = dense(w)
        tiles = -(-n // 16) * -(-k // 128)
        self.data = torch.empty(mats * tiles * 2048, dtype=w.dtype, device=w.device)
        launch("qm_tile_weight", w.device, native.act_code(w.dtype), mats, n, k, wc.data_ptr(), self.codes_ptr)

    scales_ptr = None

    @property
    def codes_ptr(self) -> int:
        return self.data.data_ptr()


class MoeWeights(SetOnce):
    """The weights of a mixture-of-experts layer, copied and laid out once for the
    kernels (an ``Mx4Weight`` is such a copy already and is kept as it is).

    ``router`` [experts, hidden] sets the activations' type; ``gate``, ``up``
    [experts, inter, hidden] and ``down`` [experts, hidden, inter] are tensors of
    that type or ``Mx4Weight``s, and so is ``shared``, the (gate, up, down) of the
    experts that every token takes (leading dimension: how many, each as wide as
    a routed one), behind the sigmoid of ``shared_router`` [hidden] when that is
    given. ``normalize``: a token's routed weights add up to 1. Its attributes do not
    change: another ``top_k`` is another ``MoeWeights``."""

    def __init__(self, router, gate, up, down, top_k: int, shared=None, shared_router=None, normalize: bool = True):
        _check_router_shape(router)
        self.router = _copy(router)
        self.experts, self.hidden = router.shape
        self.top_k, self.normalize = int(top_k), bool(normalize)
        if not 1 <= self.top_k <= min(self.experts, MAX_TOP_K):
            raise ValueError(f"top_k must be 1 to {min(self.experts, MAX_TOP_K)}, got {top_k}")
        self.is_mx4 = isinstance(gate, Mx4Weight)
        if len(gate.shape) != 3:
            raise ValueError(f"gate must be [experts, inter, hidden], got {tuple(gate.shape)}")
        self.inter = int(gate.shape[1])
        if self.inter == 0 or self.inter % BLOCK:
            raise ValueError(f"the experts' width must be a multiple of {BLOCK}, got {self.inter}")
        self.gate, self.up, self.down = self._take(self.experts, (gate, up, down), "")
        count, parts, row = 0, (None, None, None), None
        if shared is not None:
            count = int(shared[0].shape[0])
            if not 1 <= count <= MAX_SHARED:
                raise ValueError(f"1 to {MAX_SHARED} shared experts, got {count}")
            parts = self._take(count, shared, "shared ")
            if shared_router is not None:
                check_input(shared_router, "shared_router")
                if shared_router.numel() != self.hidden or shared_router.dtype != router.dtype \
                        or shared_router.device != router.device:
                    raise ValueError(f"shared_router must be [{self.hidden}] in {router.dtype} on {router.device}")
                row = _copy(shared_router.reshape(-1))
        elif shared_router is not None:
            raise ValueError("shared_router without shared experts")
        self.shared, self.shared_router = count, row
        self.s_gate, self.s_up, self.s_down = parts
        self._bind()

    def _bind(self) -> None:
        """The weights as the C ABI takes them (qm_moe_weights)."""
        mats = (self.gate, self.up, self.down, self.s_gate, self.s_up, self.s_down)
        p = [None if t is None else t.codes_ptr for t in mats]
        s = [None if t is None else t.scales_ptr for t in mats]
        self.ptrs = native.MoeWeightPtrs(self.router.data_ptr(), p[0], p[1], p[2], s[0], s[1], s[2],
                                         native.ptr(self.shared_router), p[3], p[4], p[5], s[3], s[4], s[5])
        self._ptrs_ref = ctypes.byref(self.ptrs)
        self._calls = {}

    # a copied or loaded layer has memory of its own
    def __getstate__(self):
        return {k: v for k, v in self.__dict__.items() if k not in ("ptrs", "_ptrs_ref", "_calls")}

    def __setstate__(self, state):
        self.__dict__.update(state)
        self._bind()

    def _take(self, mats: int, parts, what: str) -> list:
        out = []
        for name, t, shape in zip(("gate", "up", "down"), parts, ((mats, self.inter, self.hidden),
                                  (mats, self.inter, self.hidden), (mats, self.hidden, self.inter))):
            if tuple(t.shape) != shape:
                raise ValueError(f"{what}{name} must be {shape}, got {tuple(t.shape)}")
            if isinstance(t, Mx4Weight) != self.is_mx4:
                raise ValueError("the experts' weights must all be 4-bit or all plain")
            if t.device != self.router.device:
                raise ValueError(f"{what}{name} is on {t.device}, the router on {self.router.device}")
            if self.is_mx4:
                out.append(t)
                continue
            check_input(t, what + name)
            if t.dtype != self.router.dtype:
                raise ValueError(f"{what}{name} is {t.dtype}, the router {self.router.dtype}")
            out.append(_Tiles(t.detach()))
        return out

    @property
    def dtype(self):
        return self.router.dtype

    @property
    def device(self):
        return self.router.device

    def geom(self, rows: int) -> native.MoeGeom:
        """The geometry of a call of ``rows`` tokens (include/qwen4mix.h)."""
        return native.MoeGeom(rows, self.hidden, self.inter, self.experts, self.shared, self.top_k,
                              int(self.normalize), native.act_code(self.dtype),
                              native.QM_W_MX4 if self.is_mx4 else native.QM_W_ACT)

    def _call(self, rows: int):
        """(geometry, bytes of workspace) of a call of ``rows`` tokens, kept for the
        next of as many."""
        hit = self._calls.get(rows)
        if hit is None:
            if len(self._calls) >= 256:
                self._calls.clear()
            g = ctypes.byref(self.geom(rows))
            hit = self._calls[rows] = (g, max(native.load().qm_moe_workspace(g), 1))
        return hit


def moe(x: torch.Tensor, weights: MoeWeights) -> torch.Tensor:
    """The layer's output for x [..., hidden] (the weights' type, up to 262140 rows), in
    x's shape: the weighted sum of each token's experts plus its shared experts. A
    call's sums differ by their order between 1, 2 to 16 and more rows; its memory
    grows by (top_k + shared) hidden floats a row."""
    check_input(x, "x")
    _check_router(x, weights.router, weights.top_k)
    device = x.device
    out = torch.empty(x.shape, dtype=x.dtype, device=device)
    m = x.numel() // weights.hidden
    if m:
        xr, ldx = activation_rows(x)
        g, nbytes = weights._call(m)
        ws = torch.empty(nbytes, dtype=torch.uint8, device=device)
        launch("qm_moe", device, g, weights._ptrs_ref, xr.data_ptr(), ldx, out.data_ptr(), ws.data_ptr(), nbytes)
    return out
