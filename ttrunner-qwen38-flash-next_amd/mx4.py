"""Microscaled 4-bit weights and their products.

A weight matrix in blocks of 32 along its last dimension: a block's elements are
E2M1 (0, 0.5, 1, 1.5, 2, 3, 4, 6 and their negatives), its scale a power of two
(E8M0), 17 bytes for 32 weights. ``mx4_quantize`` makes one from a float32 or
bfloat16 tensor, ``Mx4Weight.from_codes`` from a checkpoint's codes, and
``mx4_linear`` is ``F.linear`` over it for float32 or bfloat16 activations, from
a single row to a prompt. ``Qwen4MixModel(weight_format="mx4")`` keeps a model's
projections in it, ``MoeWeights`` a mixture-of-experts layer's.

The weights live on the device in the matrix cores' operand order
(include/qwen4mix.h); everything runs in the HIP kernels of libqwen4mix.so, on
the current stream of the tensors' device. Nothing here is differentiable or
traceable: inputs that require a gradient are refused while gradients are
recorded, inputs with a tangent always, and so is any call while torch.jit.trace
or make_fx records (torch.compile breaks its graph around the calls). Autocast
casts nothing: outputs have their input's type.
"""

from __future__ import annotations

import ctypes

import torch
from torch.autograd import forward_ad

from . import native

BLOCK = 32
TILE_ROWS, TILE_K = 16, 128


_ACT = {torch.float32: native.QM_ACT_F32, torch.bfloat16: native.QM_ACT_BF16}
_raw_stream, _current_device = torch._C._cuda_getCurrentRawStream, torch._C._cuda_getDevice
_tracing_state, _dispatch_modes = torch._C._get_tracing_state, torch._C._len_torch_dispatch_stack


def refuse_recording() -> None:
    """Raise where torch records the operations of a call: it would see the output
    made and not what the kernels write into it."""
    if _tracing_state() is not None or \
            torch._C._get_dispatch_mode(torch._C._TorchDispatchModeKey.PROXY) is not None:
        raise RuntimeError("the 4-bit weights' and the experts' operators cannot be traced (torch.jit.trace, make_fx)")


def launch(name: str, device, *args) -> None:
    """The entry point ``name`` on ``args`` and the current stream of ``device``."""
    if _dispatch_modes() or _tracing_state() is not None:
        refuse_recording()
    fn, index = getattr(native.load(), name), device.index
    if index == _current_device():
        rc = fn(*args, _raw_stream(index))
    else:
        with torch.cuda.device(device):                             # kernels go to the current device
            rc = fn(*args, _raw_stream(index))
    if rc:
        native.check(name, rc)


def check_input(t: torch.Tensor, what: str) -> int:
    """The type code of a float32 or bfloat16 tensor on the GPU that loses no
    gradient or tangent here."""
    if forward_ad._current_level >= 0 and isinstance(t, torch.Tensor) and forward_ad.unpack_dual(t).tangent is not None:
        raise RuntimeError(f"{what} has a tangent, and this operator has no forward derivative")
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise ValueError(f"{what} must be a tensor on the GPU")
    if t.requires_grad and torch.is_grad_enabled():
        raise RuntimeError(f"{what} requires a gradient, and this operator has none (use torch.no_grad())")
    code = _ACT.get(t.dtype)
    return native.act_code(t.dtype) if code is None else code


def dense(t: torch.Tensor) -> torch.Tensor:
    """t, or a copy, contiguous and 16-byte aligned."""
    t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


def activation_rows(x: torch.Tensor) -> tuple[torch.Tensor, int]:
    """x [..., K] as rows [M, K] and the elements from one to the next: a view
    where the kernels can read it (whole 16-byte units), else a copy."""
    k = x.shape[-1]
    if x.is_contiguous() and x.data_ptr() % 16 == 0:
        return x, k
    rows = x.reshape(-1, k)
    if rows.stride(1) == 1 and rows.data_ptr() % 16 == 0:
        if rows.shape[0] == 1:
            return rows, k
        if rows.stride(0) >= k and rows.stride(0) * rows.element_size() % 16 == 0:
            return rows, rows.stride(0)
    return dense(rows), k


class SetOnce:
    """Attributes that are set once: calls, decoders and captured graphs keep the
    addresses and sizes that they stand for."""

    def __setattr__(self, name, value):
        if name in self.__dict__:
            raise AttributeError(f"{type(self).__name__}.{name} does not change: make a new one")
        object.__setattr__(self, name, value)

    def __delattr__(self, name):
        raise AttributeError(f"{type(self).__name__}.{name} does not change: make a new one")


class Mx4Weight(SetOnce):
    """A weight [..., n, k] in 4-bit blocks along k, laid out for the kernels.

    ``data`` holds the device tiles (uint8, 17 bytes for 32 weights of tiles of 16
    rows x 128 k), ``codes`` and ``scales`` are views of it; ``plain()`` gives them in
    a checkpoint's order, ``dequantize()`` the values they stand for. Made by
    ``mx4_quantize`` or ``from_codes``; its attributes do not change."""

    def __init__(self, data: torch.Tensor, shape):
        shape = torch.Size(shape)
        need = self._bytes(shape)
        if data.dtype != torch.uint8 or not data.is_contiguous() or data.numel() != need or data.data_ptr() % 16:
            raise ValueError(f"the tiles of {tuple(shape)} are {need} bytes (uint8, contiguous, 16-byte aligned), got "
                             f"{data.dtype} {tuple(data.shape)}")
        self._set(data, shape)

    def _set(self, data: torch.Tensor, shape: torch.Size) -> None:
        # (the codes are 16 of 17 bytes, the scales behind them)
        self.__dict__.update(data=data, shape=shape, mats=1 if len(shape) == 2 else shape[:-2].numel(),
                             code_bytes=data.numel() // 17 * 16)

    # (read from the tensor each time: a copied or loaded weight has memory of its own)
    @property
    def codes_ptr(self) -> int:
        return self.data.data_ptr()

    @property
    def scales_ptr(self) -> int:
        return self.data.data_ptr() + self.code_bytes

    @property
    def codes(self) -> torch.Tensor:
        return self.data[:self.code_bytes]

    @property
    def scales(self) -> torch.Tensor:
        return self.data[self.code_bytes:]

    @property
    def device(self):
        return self.data.device

    @staticmethod
    def _check_shape(shape) -> None:
        if len(shape) < 2 or 0 in shape:
            raise ValueError(f"a 4-bit weight needs a non-empty [..., n, k], got {tuple(shape)}")
        if shape[-1] % BLOCK:
            raise ValueError(f"the last dimension must be a multiple of {BLOCK}, got {shape[-1]}")

    @classmethod
    def _bytes(cls, shape: torch.Size) -> int:
        cls._check_shape(shape)
        n, k = shape[-2:]
        tiles = -(-n // TILE_ROWS) * -(-k // TILE_K)
        if len(shape) > 2:
            tiles *= shape[:-2].numel()
        return tiles * (TILE_ROWS * TILE_K // 32 * 17)

    @classmethod
    def _empty(cls, shape: torch.Size, device) -> "Mx4Weight":
        w = cls.__new__(cls)
        w._set(torch.empty(cls._bytes(shape), dtype=torch.uint8, device=device), shape)
        return w

    @classmethod
    def from_codes(cls, codes: torch.Tensor, scales: torch.Tensor) -> "Mx4Weight":
        """From codes uint8 [..., n, k / 2] (two elements a byte, the first in the
        low nibble; bit 3 the sign, bits 2 and 1 the exponent, bit 0 the mantissa)
        and scale bytes uint8 [..., n, k / 32] (2^(byte - 127), 255 NaN)."""
        if codes.dtype != torch.uint8 or scales.dtype != torch.uint8 or not codes.is_cuda:
            raise ValueError("codes and scales must be uint8 tensors on the GPU")
        shape = torch.Size(codes.shape[:-1] + (2 * codes.shape[-1],))
        cls._check_shape(shape)
        if scales.shape != codes.shape[:-1] + (shape[-1] // BLOCK,) or scales.device != codes.device:
            raise ValueError(f"scales must be {tuple(codes.shape[:-1]) + (shape[-1] // BLOCK,)} on {codes.device}, "
                             f"got {tuple(scales.shape)} on {scales.device}")
        w = cls._empty(shape, codes.device)
        pc, ps = dense(codes), scales.contiguous()
        launch("qm_mx4_layout", codes.device, 1, w.mats, shape[-2], shape[-1], w.codes_ptr, w.scales_ptr, pc.data_ptr(),
               ps.data_ptr())
        return w

    def plain(self) -> tuple[torch.Tensor, torch.Tensor]:
        """(codes, scales) in the order that ``from_codes`` takes."""
        lead, n, k = self.shape[:-2], self.shape[-2], self.shape[-1]
        codes = torch.empty(*lead, n, k // 2, dtype=torch.uint8, device=self.device)
        scales = torch.empty(*lead, n, k // BLOCK, dtype=torch.uint8, device=self.device)
        launch("qm_mx4_layout", self.device, 0, self.mats, n, k, self.codes_ptr, self.scales_ptr, codes.data_ptr(),
               scales.data_ptr())
        return codes, scales

    def dequantize(self, dtype: torch.dtype = torch.float32) -> torch.Tensor:
        """The values, [..., n, k]: exact in float32 and in bfloat16 (a value past
        their range is infinite)."""
        shape, device = self.shape, self.data.device
        act = native.act_code(dtype)
        out = torch.empty(shape, dtype=dtype, device=device)
        launch("qm_mx4_dequantize", device, act, self.mats, shape[-2], shape[-1], self.codes_ptr, self.scales_ptr,
               out.data_ptr())
        return out


def mx4_quantize(w: torch.Tensor) -> Mx4Weight:
    """w [..., n, k] (float32 or bfloat16 on the GPU, k a multiple of 32) in
    4-bit blocks: the scale 2^max(floor(log2 max|w|) - 2, -127), the elements to
    the nearest value, ties to the even code, magnitudes above 6 scales to 6. A
    block that holds a NaN or an infinity becomes NaN."""
    act = check_input(w, "w")
    shape, device = w.shape, w.device
    out = Mx4Weight._empty(shape, device)
    wc = dense(w)
    launch("qm_mx4_quantize", device, act, out.mats, shape[-2], shape[-1], wc.data_ptr(), out.codes_ptr, out.scales_ptr)
    return out


def mx4_linear(x: torch.Tensor, weight: Mx4Weight, sections=None):
    """F.linear(x, weight): x [..., k] -> [..., n] in x's type, summed in float.

    ``sections``, a list of row counts that add up to n, splits the rows over
    outputs of their own (the projections of one input kept as one weight): a
    list of [..., rows] tensors is returned."""
    act = check_input(x, "x")
    if not isinstance(weight, Mx4Weight) or len(weight.shape) != 2:
        raise ValueError("mx4_linear takes a 4-bit weight of one matrix [n, k]")
    n, k = weight.shape
    lead = x.shape
    if not lead or lead[-1] != k:
        raise ValueError(f"x must be [..., {k}], got {tuple(lead)}")
    device = x.device
    if device != weight.data.device:
        raise ValueError(f"x is on {device}, the weight on {weight.device}")
    lead = lead[:-1]
    m = lead.numel()
    rows = (n,)
    if sections is not None:
        rows = tuple(int(r) for r in sections)
        if min(rows, default=0) <= 0 or sum(rows) != n or len(rows) > 8:
            raise ValueError(f"sections must be 1 to 8 positive row counts that add up to {n}, got {list(rows)}")
    outs = [torch.empty(lead + (r,), dtype=x.dtype, device=device) for r in rows]
    if m:
        xr, ldx = activation_rows(x)
        if sections is None:
            seg_rows, seg_out = ctypes.byref(ctypes.c_int(n)), ctypes.byref(ctypes.c_void_p(outs[0].data_ptr()))
        else:
            seg_rows = (ctypes.c_int * len(rows))(*rows)
            seg_out = (ctypes.c_void_p * len(rows))(*[o.data_ptr() for o in outs])
        codes = weight.data.data_ptr()
        launch("qm_mx4_linear", device, act, m, n, k, codes, codes + weight.code_bytes, xr.data_ptr(), ldx, len(rows),
               seg_rows, seg_out)
    return outs[0] if sections is None else outs
