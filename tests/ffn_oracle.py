"""The FFN half of a layer and its 4-bit weights in 64 bits, from the definitions.

Every function also gives the bound its tests hold a kernel to. A float sum of n
products is off by at most n 2^-23 times the sum of their magnitudes (any order,
each addition off by up to a whole step: matrix cores may cut); a rounding to a
type by half a step, ``half(dtype)`` relative to the value.
"""

from __future__ import annotations

import torch

GRID = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]
SUM = 2.0 ** -23


def half(dtype) -> float:
    return torch.finfo(dtype).eps / 2


def mx4_encode(w):
    """(codes uint8 [..., k / 2], scales uint8 [..., k / 32]) of w, block by block."""
    flat = w.detach().double().cpu().reshape(-1, 32)
    codes = torch.zeros(flat.shape, dtype=torch.uint8)
    scales = torch.zeros(flat.shape[0], dtype=torch.uint8)
    grid = torch.tensor(GRID, dtype=torch.float64)
    for i, b in enumerate(flat):
        if not bool(torch.isfinite(b).all()):
            scales[i] = 255
            continue
        m = b.abs().max().item()
        e = -127
        if m > 0:
            e = max(torch.frexp(torch.tensor(m, dtype=torch.float64))[1].item() - 1 - 2, -127)
        scales[i] = e + 127
        d = (b.abs()[:, None] / 2.0 ** e - grid).abs()
        near = d == d.min(1, keepdim=True).values
        # the even code where two are as near
        even = near & (torch.arange(8) % 2 == 0)
        pick = torch.where(even.any(1), even.double().argmax(1), near.double().argmax(1))
        codes[i] = pick.to(torch.uint8) + 8 * torch.signbit(b).to(torch.uint8)
    packed = codes[:, 0::2] | (codes[:, 1::2] << 4)
    lead = w.shape[:-1]
    return packed.reshape(*lead, w.shape[-1] // 2), scales.reshape(*lead, w.shape[-1] // 32)


def mx4_decode(codes, scales):
    """float64 values [..., k] of codes and scale bytes."""
    grid = torch.tensor(GRID + [-v for v in GRID], dtype=torch.float64, device=codes.device)
    c = torch.stack((codes & 15, codes >> 4), -1).flatten(-2).long()
    s = torch.pow(torch.tensor(2.0, dtype=torch.float64, device=codes.device), scales.double() - 127)
    s = torch.where(scales == 255, torch.full_like(s, float("nan")), s)
    return grid[c] * s.repeat_interleave(32, -1)


def linear(x, w):
    """(x w^T, bound of a kernel's error but for the output's rounding); w float64."""
    x, w = x.double(), w.double()
    return x @ w.t(), x.shape[-1] * SUM * (x.abs() @ w.abs().t())


def route(x, router, top_k, normalize=True):
    """(ids, weights): equal logits to the lower index. Equal router rows are
    multiplied once: a library's product may sum their columns in different orders,
    and its last bits would order what is equal."""
    rows, which = torch.unique(router.double(), dim=0, return_inverse=True)
    logits = (x.double() @ rows.t())[:, which]
    order = logits.sort(dim=-1, descending=True, stable=True).indices[:, :top_k]
    w = torch.softmax(logits, -1).gather(1, order)
    return order.int(), w / w.sum(-1, keepdim=True) if normalize else w


def _ffn(x, scale, gate, up, down, dtype):
    """(scale D (silu(G x) U x), bound of its error), all rows of x."""
    x = x.double()
    a, b = x @ gate.t(), x @ up.t()
    n = x.shape[-1]
    da, db = (n * SUM * (x.abs() @ m.abs().t()) for m in (gate, up))
    s = torch.nn.functional.silu(a)
    h = scale[:, None] * s * b
    # |silu'| < 1.1; the exponential, the division and the products: 16 steps of a float
    dh = scale[:, None] * (1.1 * da * (b.abs() + db) + s.abs() * db) + (half(dtype) + 16 * SUM) * h.abs()
    inter = h.shape[-1]
    return h @ down.t(), (dh + inter * SUM * (h.abs() + dh)) @ down.abs().t()


def moe(x, router, gate, up, down, top_k, normalize=True, shared=None, shared_router=None):
    """(y, bound but for the output's rounding) of a layer with float64 weights."""
    ids, w = route(x, router, top_k, normalize)
    y = torch.zeros(x.shape, dtype=torch.float64, device=x.device)
    bound = torch.zeros_like(y)
    for e in range(gate.shape[0]):
        t, j = (ids == e).nonzero(as_tuple=True)
        if t.numel():
            o, d = _ffn(x[t], w[t, j], gate[e], up[e], down[e], x.dtype)
            y[t] += o
            bound[t] += d
    if shared is not None:
        one = torch.ones(x.shape[0], dtype=torch.float64, device=x.device)
        open_ = one if shared_router is None else torch.sigmoid(x.double() @ shared_router.double())
        for s in range(shared[0].shape[0]):
            o, d = _ffn(x, open_, *(p[s] for p in shared), x.dtype)
            y += o
            bound += d
    # the weights' exponentials and the float sum over the pairs
    pairs = top_k + (0 if shared is None else shared[0].shape[0])
    return y, bound * (1 + 2.0 ** -12) + pairs * SUM * bound / half(x.dtype)


def within(got, want, bound, dtype):
    """The largest error as a share of its bound (finite values; 1 is the limit)."""
    lim = bound + half(dtype) * want.abs() + torch.finfo(torch.float32).tiny
    return ((got.double() - want).abs() / lim).max().item()
