"""The experts and the 4-bit weights in models and decoders of other kinds than a
bf16 one with its rows side by side: float activations, rows at different positions,
pages drawn from a pool, layers of many row counts in one program.

Every expert is chosen (top_k is their number), so no choice hangs on a rounding.
Where both sides run the same kernels the results are equal bit for bit. Elsewhere
they differ by the order of sums:

* bf16 layers are held to their own bar of 2e-2;
* float DeltaNet layers to 2e-4: sums of up to 4096 products are off by some
  sqrt(4096) 2^-24 = 4e-6 each, a dozen of them one after the other, three layers;
* stacks with a QSA layer to that layer's bar of 2e-2 in float too: a decoder's plan
  and a layer call may take different attention kernels, and the cache holds K and V
  as bf16 whatever the activations (cache.py), so a value next to a border between
  two bf16 goes to the other one, a step of 2^-7 of it away.
"""

from __future__ import annotations

import os
import sys

import pytest
import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), "golden"))
import inputs as gi  # noqa: E402

from margins import rel_err  # noqa: E402

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16, F32 = torch.bfloat16, torch.float32
N_LAYERS, EXPERTS, INTER, HIDDEN = 4, 6, 64, 2048
BAR = 2e-2


def stack_weights(dtype):
    w = {}
    for l in range(N_LAYERS):
        w.update(gi.qsa_weights(l, 500 + l, dtype) if (l + 1) % 4 == 0 else gi.dn_weights(l, 500 + l, dtype))
        for kind, seed in (("attn", 600), ("ffn", 700)):
            w.update(gi.hc_weights(f"blk.{l}.hc_{kind}", seed + l, dtype))
        r, p, s = gi.rng(800 + l), f"blk.{l}.ffn_", HIDDEN ** -0.5
        for name, shape, scale in (("gate_inp", (EXPERTS, HIDDEN), s), ("gate_exps", (EXPERTS, INTER, HIDDEN), s),
                                   ("up_exps", (EXPERTS, INTER, HIDDEN), s), ("down_exps", (EXPERTS, HIDDEN, INTER), INTER ** -0.5),
                                   ("gate_shexp", (INTER, HIDDEN), s), ("up_shexp", (INTER, HIDDEN), s),
                                   ("down_shexp", (HIDDEN, INTER), INTER ** -0.5), ("gate_inp_shexp", (1, HIDDEN), s)):
            w[p + name + ".weight"] = gi.normal(r, shape, scale, dtype)
    return w


@pytest.fixture(scope="module")
def models(gpu):
    """(type, weight format) -> model, made when asked for."""
    weights, made = {}, {}

    def get(dtype, fmt):
        if dtype not in weights:
            weights[dtype] = stack_weights(dtype)
        if (dtype, fmt) not in made:
            cfg = gpu.MixConfig(num_experts_per_tok=EXPERTS)
            made[dtype, fmt] = gpu.Qwen4MixModel(cfg, gi.FakeStore(weights[dtype]), device=DEV, weight_format=fmt)
        return made[dtype, fmt]

    return get


def new_cache(qm, model, dtype, batch=1, pages="random"):
    kw = dict(seed=3) if pages == "random" else {}
    cache = qm.MixHybridCache(N_LAYERS, model.config, batch=batch, max_ctx=4096, device=DEV, dtype=dtype, page_table=pages, **kw)
    cache.ensure_allocated()
    return cache


def residuals(seed, n, rows, dtype, k=1):
    r = gi.rng(seed)
    return [gi.normal(r, (rows, k, 4 * HIDDEN)).to(dtype).to(DEV) for _ in range(n)]


def layer_methods(model, cache, x, position, layers):
    h = x
    for l in layers:
        mixed, _, inject = model._gated_residual(h, l, "attn")
        branch = (model._full_attention(mixed, l, None, None, cache, position) if model.config.is_full_attention(l)
                  else model._linear_attention(mixed, l, cache))
        h = model._reinject(h, branch, inject)
        mixed, _, inject = model._gated_residual(h, l, "ffn")
        h = model._reinject(h, model._moe(mixed, l), inject)
    return h


@pytest.mark.parametrize("fmt", ["act", "mx4"])
@pytest.mark.parametrize("layers,bar", [((0, 1, 2), 2e-4), ((0, 1, 2, 3), BAR)])
def test_float_decoder_with_experts(gpu, models, fmt, layers, bar):
    model = models(F32, fmt)
    xs = residuals(1, 4, 1, F32)
    eager = gpu.MixDecoder(model, new_cache(gpu, model, F32), layers=layers, dtype=F32, ffn=True)
    want = [eager.step_eager(x).clone() for x in xs]
    replayed = gpu.MixDecoder(model, new_cache(gpu, model, F32), layers=layers, dtype=F32, ffn=True)
    methods = new_cache(gpu, model, F32)
    for i, (x, y) in enumerate(zip(xs, want)):
        got = replayed.step(x)
        torch.cuda.synchronize()
        assert torch.equal(got, y)
        assert rel_err(y, layer_methods(model, methods, x, i, layers), bar) < bar


@pytest.mark.parametrize("fmt", ["act", "mx4"])
@pytest.mark.parametrize("k", [3, 20])
def test_float_verify_step_with_experts(gpu, models, fmt, k):
    model = models(F32, fmt)
    rows = residuals(k, 1, 1, F32, k=k)[0]
    eager = gpu.MixDecoder(model, new_cache(gpu, model, F32), dtype=F32, ffn=True).step_n(rows).clone()
    dec = gpu.MixDecoder(model, new_cache(gpu, model, F32), dtype=F32, ffn=True)
    snap = dec.snapshot()
    for _ in range(3):
        dec.restore(snap)
        got = dec.step_n_graph(rows).clone()
        torch.cuda.synchronize()
        assert torch.equal(got, eager)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("fmt", ["act", "mx4"])
def test_rows_at_different_positions_with_experts(gpu, models, dtype, fmt):
    """Two sequences of a pooled cache, four tokens and none long, in one decoder:
    as each alone."""
    model = models(dtype, fmt)
    first = residuals(11, 4, 1, dtype)
    steps = residuals(12, 3, 2, dtype)
    cache = new_cache(gpu, model, dtype, batch=2, pages="pooled")
    view = cache.slot_view(0)
    dec = gpu.MixDecoder(model, view, dtype=dtype, ffn=True)
    for x in first:
        dec.step(x)
    cache.commit_slot_view(view)
    both = gpu.MixDecoder(model, cache, dtype=dtype, positions=[4, 0], ffn=True)
    alone = [gpu.MixDecoder(model, new_cache(gpu, model, dtype), dtype=dtype, ffn=True) for _ in range(2)]
    for x in first:
        alone[0].step(x)
    for x in steps:
        got = both.step(x).clone()
        for b in range(2):
            assert rel_err(got[b:b + 1], alone[b].step(x[b:b + 1]), BAR) < BAR
    assert both.row_positions == [7, 3]


def test_two_decoders_of_one_model_share_its_experts(gpu, models):
    """Steps of two decoders in turn, each from its own graph: as each alone."""
    model = models(BF16, "mx4")
    xs = [residuals(20 + i, 4, 1, BF16) for i in range(2)]
    want = []
    for seq in xs:
        dec = gpu.MixDecoder(model, new_cache(gpu, model, BF16), ffn=True)
        want.append([dec.step(x).clone() for x in seq])
    decs = [gpu.MixDecoder(model, new_cache(gpu, model, BF16), ffn=True) for _ in xs]
    for i in range(4):
        for d, seq, ys in zip(decs, xs, want):
            got = d.step(seq[i])
            torch.cuda.synchronize()
            assert torch.equal(got, ys[i])
