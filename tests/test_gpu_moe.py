"""Routing (moe_route) and the mixture-of-experts layer (moe) against 64 bits.

The chosen experts are compared exactly (the logits are sums in double on both
sides; random ones lie far further apart than its rounding). A weight is
exp(l - max) / sum: the difference is rounded to float (|l - max| < 16 here, so
2^-20 relative), the exponential, the sum of at most 32 and the division add some
40 half steps: 2^-18 in all. Outputs are held to the bound of tests/ffn_oracle.py
and, by norm, to twice half a step of the activations' type: the hidden rows' and
the output's rounding are independent, each 0.58 half steps in the mean.
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
W_TOL = 2.0 ** -18


def normal(seed, *shape, dtype=F32, scale=1.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return (torch.randn(*shape, generator=g, device=DEV) * scale).to(dtype)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("t,e,k,h", [(1, 1, 1, 32), (1, 128, 8, 2048), (2, 5, 5, 96), (3, 64, 32, 160), (9, 130, 6, 512),
                                     (17, 1024, 32, 64), (64, 60, 4, 2080), (333, 256, 10, 256), (1000, 16, 2, 1024)])
@pytest.mark.parametrize("normalize", [True, False])
def test_route_matches_f64(gpu, dtype, t, e, k, h, normalize):
    x, r = normal(t + e, t, h, dtype=dtype), normal(h, e, h, dtype=dtype, scale=h ** -0.5)
    ids, w = gpu.moe_route(x, r, k, normalize)
    want_ids, want_w = fo.route(x, r, k, normalize)
    assert ids.dtype == torch.int32 and w.dtype == F32 and ids.shape == (t, k)
    assert torch.equal(ids, want_ids)
    rel = ((w.double() - want_w).abs() / want_w).max().item()
    assert record("rel", rel, W_TOL) < W_TOL


@pytest.mark.parametrize("t", [1, 6, 70])
def test_route_ties_and_bad_values(gpu, t):
    h, e = 64, 12
    x = normal(1, t, h, dtype=BF16)
    r = normal(2, e, h, dtype=BF16)
    r[3] = r[7] = r[9]                                             # equal logits, always
    ids, w = gpu.moe_route(x, r, e)
    order = ids[0].tolist()
    for row in ids.tolist():
        assert row.index(3) + 1 == row.index(7) and row.index(7) + 1 == row.index(9)
        assert sorted(row) == list(range(e))
    assert order == fo.route(x, r, e)[0][0].tolist()
    zero = torch.zeros_like(x)
    ids, w = gpu.moe_route(zero, r, 4)                             # every logit equal
    assert ids.tolist() == [[0, 1, 2, 3]] * t and bool((w == 0.25).all())
    ids, w = gpu.moe_route(-zero, r, 4)
    assert ids.tolist() == [[0, 1, 2, 3]] * t
    x2 = x.clone()
    x2[0, 5] = float("nan")
    ids2, w2 = gpu.moe_route(x2, r, 5)
    assert ids2[0].tolist() == [0, 1, 2, 3, 4] and bool(w2[0].isnan().all())
    ids, w = gpu.moe_route(x, r, 5)
    assert torch.equal(ids2[1:], ids[1:]) and torch.equal(w2[1:], w[1:])
    r2 = r.clone()
    r2[8, 0] = float("nan")
    ids3, w3 = gpu.moe_route(x, r2, 2)
    assert bool((ids3[:, 0] == 8).all()) and bool(w3.isnan().all())


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("t,e,k", [(1, 50, 6), (5, 100, 8), (1, 300, 32), (20, 700, 3)])
def test_route_magnitudes_and_many_equal_logits(gpu, dtype, t, e, k):
    """Logits far below and above float's range, and more equal ones than a wave's lanes."""
    h = 160
    x, r = normal(t, t, h, dtype=dtype), normal(e, e, h, dtype=dtype, scale=h ** -0.5)
    for scale in (2.0 ** -100, 2.0 ** 100):
        xs, rs = x * scale, r * scale                               # powers of two: the same order
        ids, w = gpu.moe_route(xs, rs, k)
        assert torch.equal(ids, fo.route(xs, rs, k)[0]) and torch.equal(ids, fo.route(x, r, k)[0])
        assert bool((w.sum(-1) - 1).abs().max() < 2.0 ** -20)
    big = (x.double() @ r.double().t()).argmax(-1)[0].item()
    r[::2] = r[big]                                                 # half of the experts lead the first token
    ids, w = gpu.moe_route(x, r, k)
    assert torch.equal(ids, fo.route(x, r, k)[0])
    ids, w = gpu.moe_route(torch.zeros_like(x), r, k)
    assert ids.tolist() == [list(range(k))] * t and torch.equal(w, torch.full_like(w, w[0, 0].item()))


def test_route_does_not_depend_on_the_rows_beside(gpu):
    x, r = normal(5, 300, 512, dtype=BF16), normal(6, 96, 512, dtype=BF16, scale=0.05)
    ids, w = gpu.moe_route(x, r, 7)
    for lo, hi in ((0, 1), (4, 6), (10, 27), (100, 260)):
        part_ids, part_w = gpu.moe_route(x[lo:hi], r, 7)
        assert torch.equal(part_ids, ids[lo:hi])
        assert ((part_w.double() / w[lo:hi].double() - 1).abs().max().item()) < W_TOL


# Many rows: the logits come from the matrix cores and only close ones are summed
# again. A logit is then off by at most B = (129 2^-23) |x| |R[e]|; a weight, the
# exponential of a difference over a sum of such, by 4 B relative. Over all weights
# (|x| = h^1/2, |R[e]| = 1): each of a block's 128 additions is off by less than a
# step of a partial sum whose mean is 0.67 (128 / h)^1/2 at its end, all in one
# direction at worst, h / 128 blocks: 4.1e-5 a logit at h = 2080, 2^-14 for the
# difference of two.
MANY = [(500, 130, 8, 2080), (130, 1024, 32, 1056), (1700, 60, 4, 1024), (3300, 16, 2, 2048), (1001, 257, 1, 416)]


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("t,e,k,h", MANY)
@pytest.mark.parametrize("normalize", [True, False])
def test_route_many_rows(gpu, dtype, t, e, k, h, normalize):
    t = t if dtype == BF16 else 5 * t
    assert t * e * h > (1e8 if dtype == BF16 else 4.5e8)
    x, r = normal(t + e, t, h, dtype=dtype), normal(h, e, h, dtype=dtype, scale=h ** -0.5)
    ids, w = gpu.moe_route(x, r, k, normalize)
    want_ids, want_w = fo.route(x, r, k, normalize)
    assert torch.equal(ids, want_ids)
    rel = (w.double() - want_w).abs() / want_w
    lim = W_TOL + 4 * 129 * 2.0 ** -23 * x.double().norm(dim=-1) * r.double().norm(dim=-1).max()
    assert record("bound", (rel / lim[:, None]).max().item(), 1.0) <= 1.0
    rms = rel.square().mean().sqrt().item()
    assert record("rms", rms, 2.0 ** -14) < 2.0 ** -14
    for lo, hi in ((0, 1), (63, 66), (t - 20, t)):                  # as the same rows alone
        assert torch.equal(gpu.moe_route(x[lo:hi], r, k, normalize)[0], ids[lo:hi])
    base = torch.zeros(t, h + 64, dtype=dtype, device=DEV)
    base[:, 32:32 + h] = x                                          # rows apart
    ids2, w2 = gpu.moe_route(base[:, 32:32 + h], r, k, normalize)
    assert torch.equal(ids2, ids) and torch.equal(w2, w)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("copies", [3, 40, 150])
def test_route_many_rows_close_logits(gpu, dtype, copies):
    """Router rows a last bit apart (the order takes sums in double) and equal ones."""
    t, e, h, k = 600 if dtype == BF16 else 2600, 160, 1184, 12
    x = normal(1, t, h, dtype=dtype)
    r = normal(2, e, h, dtype=dtype, scale=h ** -0.5)
    near = torch.randperm(e, generator=torch.Generator().manual_seed(3))[:copies].tolist()
    r[near] = r[near[0]].clone()
    for i, n in enumerate(near):
        if i % 3:                                                   # every third stays equal
            r[n, i] += r[n, i] * torch.finfo(dtype).eps
    x += 3 * r[near[0]]
    ids, w = gpu.moe_route(x, r, k)
    assert torch.equal(ids, fo.route(x, r, k)[0])
    assert torch.equal(gpu.moe_route(x[77:80], r, k)[0], ids[77:80])
    assert bool((w[:, :-1] >= w[:, 1:]).all())


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_route_many_rows_ties_magnitudes_and_bad_values(gpu, dtype):
    t, e, h, k = 700 if dtype == BF16 else 3100, 96, 1632, 6
    r = normal(2, e, h, dtype=dtype, scale=h ** -0.5)
    x = normal(1, t, h, dtype=dtype)
    x *= torch.logspace(-38, 17, t, device=DEV).to(dtype)[:, None]
    x[5] = 0
    x[6] = 0
    x[6, 9] = torch.finfo(dtype).tiny
    ids, w = gpu.moe_route(x, r, k)
    want = fo.route(x, r, k)[0]
    assert torch.equal(ids, want) and ids[5].tolist() == list(range(k))
    assert bool((w.sum(-1) - 1).abs().max() < 2.0 ** -20) and bool((w[5] == w[5, 0]).all())
    small = normal(4, e, h, dtype=dtype, scale=1e-30)               # products below float's range
    assert torch.equal(gpu.moe_route(x, small, k)[0], fo.route(x, small, k)[0])
    zero = torch.zeros_like(x)
    ids0, w0 = gpu.moe_route(zero, r, k)
    assert ids0.tolist() == [list(range(k))] * t and torch.equal(w0, torch.full_like(w0, w0[0, 0].item()))
    x = normal(1, t, h, dtype=dtype)
    clean, cw = gpu.moe_route(x, r, k)
    bad = x.clone()
    bad[0, 3], bad[64, h - 1], bad[t - 1, 0], bad[300] = float("nan"), float("inf"), float("-inf"), float("nan")
    ids, w = gpu.moe_route(bad, r, k)
    hit = [0, 64, 300, t - 1]
    for i in hit:
        alone_ids, alone_w = gpu.moe_route(bad[i:i + 1], r, k)
        assert torch.equal(ids[i:i + 1], alone_ids) and bool(w[i].isnan().all()) and bool(alone_w.isnan().all())
    keep = [i for i in range(t) if i not in hit]
    assert torch.equal(ids[keep], clean[keep]) and torch.equal(w[keep], cw[keep])
    r2 = r.clone()
    r2[70, 1] = float("nan")
    ids, w = gpu.moe_route(x, r2, k)
    assert bool((ids[:, 0] == 70).all()) and bool(w.isnan().all())


def layer(qm, seed, e, h, i, shared, top_k, fmt, dtype, gated=True, normalize=True, bias=None):
    """(MoeWeights, the oracle's arguments)."""
    router = normal(seed, e, h, dtype=dtype, scale=h ** -0.5)
    mats = [normal(seed + 1, e, i, h, dtype=dtype, scale=h ** -0.5), normal(seed + 2, e, i, h, dtype=dtype, scale=h ** -0.5),
            normal(seed + 3, e, h, i, dtype=dtype, scale=i ** -0.5)]
    sh = None
    if shared:
        sh = [normal(seed + 4, shared, i, h, dtype=dtype, scale=h ** -0.5),
              normal(seed + 5, shared, i, h, dtype=dtype, scale=h ** -0.5),
              normal(seed + 6, shared, h, i, dtype=dtype, scale=i ** -0.5)]
    if bias is not None:
        mats = bias(mats)
    gate_row = normal(seed + 7, h, dtype=dtype, scale=h ** -0.5) if shared and gated else None
    if fmt == "mx4":
        mats = [qm.mx4_quantize(m) for m in mats]
        sh = None if sh is None else [qm.mx4_quantize(m) for m in sh]
        values = [m.dequantize().double() for m in mats]
        sh_values = None if sh is None else [m.dequantize().double() for m in sh]
    else:
        values, sh_values = [m.double() for m in mats], None if sh is None else [m.double() for m in sh]
    w = qm.MoeWeights(router, *mats, top_k=top_k, shared=sh, shared_router=gate_row, normalize=normalize)
    return w, dict(router=router, gate=values[0], up=values[1], down=values[2], top_k=top_k, normalize=normalize,
                   shared=sh_values, shared_router=gate_row)


def check(got, x, args):
    want, bound = fo.moe(x, **args)
    assert got.shape == x.shape and got.dtype == x.dtype
    assert record("bound", fo.within(got, want, bound, x.dtype), 1.0) <= 1.0
    rel = ((got.double() - want).norm() / want.norm()).item()
    lim = 2 * fo.half(x.dtype) if x.dtype == BF16 else 2 ** -19
    assert record("norm", rel, lim) < lim


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("fmt", ["plain", "mx4"])
@pytest.mark.parametrize("t,e,k,h,i,shared", [(1, 4, 2, 64, 32, 0), (1, 16, 8, 2048, 512, 1), (2, 7, 3, 96, 160, 2),
                                              (4, 32, 8, 512, 352, 1), (5, 3, 3, 160, 96, 0), (9, 24, 8, 1024, 256, 1),
                                              (16, 8, 2, 256, 64, 3), (17, 9, 1, 288, 128, 1), (33, 40, 6, 128, 96, 0),
                                              (70, 12, 4, 544, 224, 1), (260, 6, 3, 256, 128, 1), (300, 64, 8, 128, 64, 2)])
def test_moe_matches_f64(gpu, dtype, fmt, t, e, k, h, i, shared):
    print(f"moe {dtype} {fmt} t={t} e={e} k={k} h={h} i={i} shared={shared}", flush=True)
    w, args = layer(gpu, t + e, e, h, i, shared, k, fmt, dtype, gated=t % 2 == 1, normalize=t % 3 != 0)
    x = normal(t, t, h, dtype=dtype)
    check(gpu.moe(x, w), x, args)


# the borders between the kernels: 16 and 17 tokens; row tiles of 64 and 128; experts'
# lists by the choosing waves and apart, over one round of choices and several;
# weights read once; logits by matrix cores; the largest top_k, experts and shared
@pytest.mark.parametrize("fmt", ["plain", "mx4"])
@pytest.mark.parametrize("t,e,k,h,i,shared", [(16, 24, 4, 288, 160, 1), (17, 24, 4, 288, 160, 1), (300, 8, 2, 160, 96, 1),
                                              (300, 16, 2, 160, 96, 1), (1100, 4, 2, 160, 96, 1), (3000, 32, 6, 64, 32, 0),
                                              (290, 24, 2, 96, 64, 0), (280, 24, 2, 96, 64, 1), (1700, 60, 4, 1056, 32, 1),
                                              (16, 1024, 32, 32, 32, 1), (40, 1024, 32, 32, 32, 0), (3, 32, 32, 64, 32, 32),
                                              (20, 32, 32, 64, 32, 32), (16, 1, 1, 96, 32, 0), (90, 1, 1, 96, 32, 0)])
def test_moe_borders(gpu, fmt, t, e, k, h, i, shared):
    print(f"moe {fmt} t={t} e={e} k={k} h={h} i={i} shared={shared}", flush=True)
    w, args = layer(gpu, t + e, e, h, i, shared, k, fmt, BF16, normalize=t % 2 == 0)
    x = normal(t, t, h, dtype=BF16)
    check(gpu.moe(x, w), x, args)


@pytest.mark.parametrize("fmt", ["plain", "mx4"])
def test_a_copied_layer_has_its_own_memory(gpu, fmt):
    w, args = layer(gpu, 5, 6, 96, 64, 1, 2, fmt, BF16)
    x = normal(6, 20, 96, dtype=BF16)
    want = gpu.moe(x, w)
    for other in (copy.deepcopy(w), pickle.loads(pickle.dumps(w))):
        assert torch.equal(gpu.moe(x, other), want)
        for t in (other.down, other.s_down):
            t.data.zero_()
        assert not bool(gpu.moe(x, other).any()) and torch.equal(gpu.moe(x, w), want)


@pytest.mark.parametrize("fmt", ["plain", "mx4"])
@pytest.mark.parametrize("t", [1, 9, 60, 400])
def test_calls_on_two_streams_at_once(gpu, fmt, t):
    w, args = layer(gpu, 21, 16, 256, 128, 1, 4, fmt, BF16)
    xs = [normal(60 + i, t, 256, dtype=BF16) for i in range(2)]
    want = [gpu.moe(x, w) for x in xs]
    streams = [torch.cuda.Stream() for _ in xs]
    got = [[], []]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(6):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(gpu.moe(xs[i], w))
    torch.cuda.synchronize()
    assert all(torch.equal(g, y) for gs, y in zip(got, want) for g in gs)


@pytest.mark.parametrize("fmt", ["plain", "mx4"])
@pytest.mark.parametrize("t", [1, 3, 12, 64, 500])
def test_all_tokens_on_few_experts(gpu, fmt, t):
    """Every token on the same two experts: the others have no rows."""
    w, args = layer(gpu, 3, 20, 128, 64, 1, 2, fmt, BF16)
    x = normal(t, t, 128, dtype=BF16, scale=0.1)
    x += (args["router"][5] + args["router"][17]) * 8
    got = gpu.moe(x, w)
    assert set(gpu.moe_route(x, args["router"], 2)[0].flatten().tolist()) == {5, 17}
    check(got, x, args)


@pytest.mark.parametrize("fmt", ["plain", "mx4"])
@pytest.mark.parametrize("t", [1, 2, 8, 14, 40, 200])
def test_bad_values_stay_with_their_tokens(gpu, fmt, t):
    """A token with a NaN is NaN and leaves the others alone; an expert with
    infinite or NaN weights reaches only the tokens that chose it."""
    e, k = 10, 2

    def spoil(mats):
        mats[0][4, 0, 0], mats[2][6, 1, 1], mats[1][6, 2, 2] = float("nan"), float("inf"), float("inf")
        return mats

    w, args = layer(gpu, 8, e, 96, 64, 1, k, fmt, BF16, bias=spoil)
    x = normal(t + 50, t, 96, dtype=BF16)
    ids = gpu.moe_route(x, args["router"], k)[0]
    got = gpu.moe(x, w)
    hit = ((ids == 4) | (ids == 6)).any(-1)
    assert torch.equal(got.isfinite().all(-1), ~hit)
    x2 = x.clone()
    x2[t // 2, 7] = float("nan")
    got2 = gpu.moe(x2, w)
    assert bool(got2[t // 2].isnan().all())
    keep = [r for r in range(t) if r != t // 2 and not bool(hit[r])]
    assert torch.equal(got2[keep], got[keep])


@pytest.mark.parametrize("t", [1, 4, 30, 200])
def test_strides_shapes_streams_and_repeats(gpu, t):
    w, args = layer(gpu, 11, 16, 128, 96, 1, 4, "mx4", BF16)
    base = normal(t, t, 300, dtype=BF16)
    x = base[:, 8:136]                                             # rows 600 bytes apart: copied
    want = gpu.moe(x.contiguous(), w)
    check(want, x.contiguous(), args)
    assert torch.equal(gpu.moe(x, w), want)
    wide = normal(t, t, 304, dtype=BF16)[:, 16:144]                # rows 608 bytes apart: read in place
    assert torch.equal(gpu.moe(wide, w), gpu.moe(wide.contiguous(), w))
    assert torch.equal(gpu.moe(x.reshape(1, t, 1, 128), w).reshape(t, 128), want)
    assert gpu.moe(x[:0], w).shape == (0, 128)
    assert all(torch.equal(gpu.moe(x, w), want) for _ in range(3))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = gpu.moe(x, w)
    here = gpu.moe(x, w)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(other, want) and torch.equal(here, want)


@pytest.mark.parametrize("t", [1, 7, 90])
def test_graph_replays(gpu, t):
    w, args = layer(gpu, 12, 16, 128, 96, 1, 4, "plain", BF16)
    xs = [normal(30 + s, t, 128, dtype=BF16) for s in range(4)]
    want = [gpu.moe(x, w) for x in xs]
    static = xs[0].clone()
    graphs = []
    for _ in range(2):                                             # two graphs of the same weights
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            ids, weights = gpu.moe_route(static, args["router"], 4)
            out = gpu.moe(static, w)
        graphs.append((g, out, ids))
    for x, y in zip(xs, want):
        static.copy_(x)
        for g, _, _ in graphs:
            g.replay()
        gpu.moe(xs[1], w)
        torch.cuda.synchronize()
        for _, out, ids in graphs:
            assert torch.equal(out, y) and torch.equal(ids, gpu.moe_route(x, args["router"], 4)[0])


@pytest.mark.parametrize("fmt", ["plain", "mx4"])
@pytest.mark.parametrize("t,e,k,h,i", [(1, 16, 8, 256, 1536), (4, 64, 8, 544, 480), (13, 40, 6, 2048, 288)])
def test_output_tiles_of_two_workgroups(gpu, fmt, t, e, k, h, i):
    """Few tokens whose down products are long: two workgroups an output tile, the
    last of which adds. Repeated, on two streams at once, and replayed."""
    w, args = layer(gpu, t + i, e, h, i, 1, k, fmt, BF16)
    xs = [normal(70 + s, t, h, dtype=BF16) for s in range(3)]
    want = [gpu.moe(x, w) for x in xs]
    for x, y in zip(xs, want):
        check(y, x, args)
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(5):
        for s, x in zip(streams, xs):
            with torch.cuda.stream(s):
                got.append(gpu.moe(x, w))
    torch.cuda.synchronize()
    assert all(torch.equal(y, want[n % 2]) for n, y in enumerate(got))
    static = xs[0].clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = gpu.moe(static, w)
    for x, y in zip(xs, want):
        static.copy_(x)
        graph.replay()
        gpu.moe(xs[0], w)
        torch.cuda.synchronize()
        assert torch.equal(out, y)


def test_refusals(gpu):
    r = normal(1, 8, 64, dtype=BF16)
    gate, up, down = normal(2, 8, 32, 64, dtype=BF16), normal(3, 8, 32, 64, dtype=BF16), normal(4, 8, 64, 32, dtype=BF16)
    x = normal(5, 3, 64, dtype=BF16)
    with pytest.raises(ValueError, match="top_k"):
        gpu.moe_route(x, r, 9)
    with pytest.raises(ValueError, match="top_k"):
        gpu.moe_route(x, r, 0)
    with pytest.raises(ValueError, match="router"):
        gpu.moe_route(x.float(), r, 2)
    with pytest.raises(ValueError, match="hidden"):
        gpu.moe_route(normal(1, 3, 40, dtype=BF16), normal(1, 8, 40, dtype=BF16), 2)
    with pytest.raises(ValueError, match="1 to 1024"):
        gpu.moe_route(x, normal(1, 1025, 64, dtype=BF16), 2)
    with pytest.raises(ValueError, match="up must be"):
        gpu.MoeWeights(r, gate, up[:, :, :32], down, 2)
    with pytest.raises(ValueError, match="4-bit or all plain"):
        gpu.MoeWeights(r, gate, up, gpu.mx4_quantize(down), 2)
    with pytest.raises(ValueError, match="float32"):
        gpu.MoeWeights(r, gate, up, down.float(), 2)
    with pytest.raises(ValueError, match="shared gate must be"):
        gpu.MoeWeights(r, gate, up, down, 2, shared=(gate[:1, :16], up[:1], down[:1]))
    with pytest.raises(ValueError, match="without shared"):
        gpu.MoeWeights(r, gate, up, down, 2, shared_router=r[0])
    w = gpu.MoeWeights(r, gate, up, down, 2)
    with pytest.raises(ValueError, match=r"\[\.\.\., 64\]"):
        gpu.moe(x[:, :32], w)
    with pytest.raises(RuntimeError, match="gradient"):
        gpu.moe(x.requires_grad_(), w)
