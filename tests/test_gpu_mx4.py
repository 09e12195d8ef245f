"""4-bit weights (mx4_quantize, Mx4Weight, mx4_linear) against 64-bit restatements.

Codes and scales are compared bit for bit, products with the bound of
tests/ffn_oracle.py (a float sum of k exact products, one rounding to the
activations' type) and, over a whole output, with a norm: independent roundings
of half a step have 0.58 of it in the mean, so twice half a step is ample.
"""

from __future__ import annotations

import copy
import pickle

import pytest
import torch

import ffn_oracle as fo
from margins import record

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16, F32 = torch.bfloat16, torch.float32


def normal(seed, *shape, dtype=F32, scale=1.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return (torch.randn(*shape, generator=g, device=DEV) * scale).to(dtype)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("shape", [(1, 32), (16, 128), (17, 160), (3, 5, 96), (33, 416)])
def test_quantize_matches_definition(gpu, dtype, shape):
    w = normal(sum(shape), *shape, dtype=dtype, scale=0.3)
    w.view(-1, 32)[::3] *= 2.0 ** 20
    q = gpu.mx4_quantize(w)
    codes, scales = q.plain()
    want_c, want_s = fo.mx4_encode(w)
    assert torch.equal(scales.cpu(), want_s)
    assert torch.equal(codes.cpu(), want_c)
    for dt in (F32, BF16):
        assert torch.equal(q.dequantize(dt).double().cpu(), fo.mx4_decode(want_c, want_s))
    # the plain order goes back into the same tiles
    again = gpu.Mx4Weight.from_codes(codes, scales)
    assert torch.equal(again.codes, q.codes) and torch.equal(again.scales, q.scales)


def test_quantize_ties_borders_and_extremes(gpu):
    mags = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, 7.0, 7.9921875, 4.0, 0.0])
    rows = []
    for e in (-149, -140, -127, -126, -120, -3, 0, 1, 100, 124):
        b = torch.zeros(32)
        b[:12] = (mags.double() * 2.0 ** e).float()
        b[12:24] = -b[:12]
        rows.append(b)
    rows += [torch.zeros(32), -torch.zeros(32)]
    w = torch.stack(rows).to(DEV)
    codes, scales = gpu.mx4_quantize(w).plain()
    want_c, want_s = fo.mx4_encode(w)
    assert torch.equal(scales.cpu(), want_s) and torch.equal(codes.cpu(), want_c)


def test_quantize_nan_and_infinite_blocks(gpu):
    w = normal(3, 4, 96)
    w[0, 5], w[1, 40], w[2, 95] = float("nan"), float("inf"), float("-inf")
    got = gpu.mx4_quantize(w).dequantize()
    bad = got.view(4, 3, 32).isnan()
    assert torch.equal(bad.all(-1), bad.any(-1))
    assert bad.any(-1).tolist() == [[True, False, False], [False, True, False], [False, False, True], [False] * 3]


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("m,n,k", [(1, 16, 32), (1, 33, 96), (2, 100, 2048), (5, 1, 128), (7, 250, 4096), (16, 48, 160),
                                   (17, 64, 256), (31, 130, 544), (64, 512, 2048), (100, 77, 96), (129, 300, 1056),
                                   (257, 1000, 640)])
def test_linear_matches_f64(gpu, dtype, m, n, k):
    q = gpu.mx4_quantize(normal(n, n, k, scale=k ** -0.5))
    x = normal(m + k, m, k, dtype=dtype)
    want, bound = fo.linear(x, q.dequantize(F32))
    got = gpu.mx4_linear(x, q)
    assert got.shape == (m, n) and got.dtype == dtype
    assert record("bound", fo.within(got, want, bound, dtype), 1.0) <= 1.0
    if m * n >= 64:
        rel = ((got.double() - want).norm() / want.norm()).item()
        lim = 2 * fo.half(dtype) if dtype == BF16 else 2 ** -19      # float sums: some dozens of half steps
        assert record("norm", rel, lim) < lim


@pytest.mark.parametrize("m", [1, 3, 20, 200])
def test_linear_sections_shapes_and_strides(gpu, m):
    q = gpu.mx4_quantize(normal(1, 75, 192, dtype=BF16))
    base = normal(2, m, 400, dtype=BF16)
    x = base[:, 8:200]                                              # rows 800 bytes apart, 16-byte aligned
    whole = gpu.mx4_linear(x.contiguous(), q)
    parts = gpu.mx4_linear(x, q, sections=[32, 1, 42])
    assert [p.shape[-1] for p in parts] == [32, 1, 42]
    assert torch.equal(torch.cat(parts, -1), whole)
    odd = base[:, 3:195]                                            # not 16-byte aligned: copied
    assert torch.equal(gpu.mx4_linear(odd, q), gpu.mx4_linear(odd.contiguous(), q))
    one = x[:1].expand(m, 192)                                      # stride 0
    assert torch.equal(gpu.mx4_linear(one, q), gpu.mx4_linear(one.contiguous(), q))
    turned = normal(4, 192, m, dtype=BF16).t()
    assert torch.equal(gpu.mx4_linear(turned, q), gpu.mx4_linear(turned.contiguous(), q))
    assert gpu.mx4_linear(x.reshape(1, m, 1, 192), q).shape == (1, m, 1, 75)
    assert gpu.mx4_linear(x[:0], q).shape == (0, 75)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("m", [1, 9, 40, 150])
def test_linear_keeps_bad_values_to_their_rows(gpu, dtype, m):
    k = 224                                                         # a last tile that is partly past k
    q = gpu.mx4_quantize(normal(5, 70, k))
    x = normal(6, m, k, dtype=dtype)
    clean = gpu.mx4_linear(x, q)
    x[0, k - 1] = float("nan")
    if m > 2:
        x[2, 0] = float("inf")
    got = gpu.mx4_linear(x, q)
    assert bool(got[0].isnan().all())
    if m > 2:
        assert not bool(got[2].isfinite().any()) or bool((q.dequantize()[:, 0] == 0).any())
    keep = [i for i in range(m) if i not in (0, 2)]
    assert torch.equal(got[keep], clean[keep])
    w = normal(7, 70, k)
    w[11, 200] = float("nan")
    bad = gpu.mx4_linear(normal(6, m, k, dtype=dtype), gpu.mx4_quantize(w))
    assert bool(bad[:, 11].isnan().all()) and bool(bad[:, :11].isfinite().all()) and bool(bad[:, 12:].isfinite().all())


# One size for each tiling that many rows can take (the workgroups that a tile
# leaves decide), at the smallest k that still ends inside a tile of 128.
TILINGS = [(40, 300), (60, 1300), (40, 4090), (60, 4090), (100, 4090), (170, 4090), (300, 4090), (600, 4090),
           (700, 4090), (1030, 4090), (1600, 4090), (2000, 1000)]


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("m,n", TILINGS)
@pytest.mark.parametrize("k", [160, 416])
def test_linear_tilings(gpu, dtype, m, n, k):
    q = gpu.mx4_quantize(normal(n, n, k, dtype=dtype, scale=k ** -0.5))
    base = normal(m + k, m, k + 64, dtype=dtype)
    x = base[:, 32:32 + k]                                          # rows apart
    want, bound = fo.linear(x, q.dequantize(F32))
    got = gpu.mx4_linear(x, q)
    assert record("bound", fo.within(got, want, bound, dtype), 1.0) <= 1.0
    lim = 2 * fo.half(dtype) if dtype == BF16 else 2 ** -19
    assert record("norm", ((got.double() - want).norm() / want.norm()).item(), lim) < lim
    parts = gpu.mx4_linear(x, q, sections=[17, n - 19, 2])
    assert torch.equal(torch.cat(parts, -1), got)
    bad = x.clone()
    bad[m // 2, k - 1], bad[m - 1, 0] = float("nan"), float("inf")
    spoilt = gpu.mx4_linear(bad, q)
    assert bool(spoilt[m // 2].isnan().all()) and not bool(spoilt[m - 1].isfinite().all())
    keep = torch.arange(m, device=DEV)
    keep = keep[(keep != m // 2) & (keep != m - 1)]
    assert torch.equal(spoilt[keep], got[keep])


def test_linear_float_activations_keep_their_bits(gpu):
    """A float activation enters as three bf16 parts: against a weight of ones in
    one block, sums of few terms are exact."""
    w = torch.zeros(16, 32, device=DEV)
    w[torch.arange(16), torch.arange(16)] = 1.0
    x = normal(8, 6, 32) * torch.logspace(-30, 30, 6, device=DEV)[:, None]
    got = gpu.mx4_linear(x, gpu.mx4_quantize(w))
    assert torch.equal(got, x[:, :16])


def test_linear_on_a_side_stream_and_in_a_graph(gpu):
    q = gpu.mx4_quantize(normal(9, 300, 512, dtype=BF16))
    xs = [normal(20 + i, 5, 512, dtype=BF16) for i in range(4)]
    want = [gpu.mx4_linear(x, q) for x in xs]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = [gpu.mx4_linear(x, q) for x in xs]
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    static = xs[0].clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = gpu.mx4_linear(static, q)
    for x, w in zip(xs, want):
        static.copy_(x)
        graph.replay()
        gpu.mx4_linear(x, q)                                        # eager work between the replays
        torch.cuda.synchronize()
        assert torch.equal(out, w)


def test_a_copied_and_a_saved_weight_have_their_own_memory(gpu):
    q = gpu.mx4_quantize(normal(3, 40, 160, dtype=BF16))
    x = normal(4, 5, 160, dtype=BF16)
    want = gpu.mx4_linear(x, q)
    for other in (copy.deepcopy(q), pickle.loads(pickle.dumps(q))):
        assert other.data.data_ptr() != q.data.data_ptr()
        assert other.codes_ptr == other.codes.data_ptr() and other.scales_ptr == other.scales.data_ptr()
        other.data.zero_()                                          # leaves the first alone
        assert not bool(gpu.mx4_linear(x, other).any())
        assert torch.equal(gpu.mx4_linear(x, q), want)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("m", [1, 40, 300])
def test_linear_with_subnormal_weights_and_activations(gpu, dtype, m):
    """Scale byte 0 (elements from 2^-128) and activations below float's normal range."""
    w = torch.zeros(64, 64, device=DEV)
    w[torch.arange(64), torch.arange(64)] = 3 * 2.0 ** -127 if dtype == BF16 else 1.0
    x = normal(5, m, 64, dtype=dtype)
    if dtype == F32:
        x *= 2.0 ** -120
    q = gpu.mx4_quantize(w)
    want = x.double() * q.dequantize().double().diagonal()
    got = gpu.mx4_linear(x, q).double()
    # One product a sum: the output's rounding, for bf16 a step of its subnormals at
    # most. A float's three bf16 parts reach down to bf16's smallest subnormal, 2^-133:
    # x = hi + mid + lo + r, each part cut towards zero at its eighth bit or at 2^-133,
    # whichever is more, so |r| < 2^-133, and the weight is 1.
    assert bool(((got - want).abs() <= fo.half(dtype) * want.abs() + 2.0 ** -133).all())


@pytest.mark.parametrize("m", [3, 40, 700])
def test_linear_calls_on_two_streams_at_once(gpu, m):
    q = gpu.mx4_quantize(normal(9, 2000, 512, dtype=BF16))
    xs = [normal(40 + i, m, 512, dtype=BF16) for i in range(2)]
    want = [gpu.mx4_linear(x, q) for x in xs]
    streams = [torch.cuda.Stream() for _ in xs]
    got = [[], []]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(6):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(gpu.mx4_linear(xs[i], q))
    torch.cuda.synchronize()
    assert all(torch.equal(g, w) for gs, w in zip(got, want) for g in gs)


def test_refusals(gpu):
    q = gpu.mx4_quantize(normal(1, 8, 64))
    x = normal(2, 3, 64)
    with pytest.raises(ValueError, match="multiple of 32"):
        gpu.mx4_quantize(normal(1, 8, 48))
    with pytest.raises(ValueError, match="n, k"):
        gpu.mx4_quantize(normal(1, 64))
    with pytest.raises(ValueError, match="non-empty"):
        gpu.mx4_quantize(normal(1, 0, 64))
    with pytest.raises(gpu.native.QmError, match="dtype"):
        gpu.mx4_quantize(normal(1, 8, 64).half())
    with pytest.raises(ValueError, match=r"\[\.\.\., 64\]"):
        gpu.mx4_linear(x[:, :32], q)
    with pytest.raises(ValueError, match="sections"):
        gpu.mx4_linear(x, q, sections=[4, 5])
    with pytest.raises(ValueError, match="one matrix"):
        gpu.mx4_linear(x, gpu.mx4_quantize(normal(1, 2, 8, 64)))
    with pytest.raises(RuntimeError, match="gradient"):
        gpu.mx4_linear(x.requires_grad_(), q)
    with torch.no_grad():
        gpu.mx4_linear(x, q)
    codes, scales = q.plain()
    with pytest.raises(ValueError, match="scales must be"):
        gpu.Mx4Weight.from_codes(codes, scales[:, :1])
