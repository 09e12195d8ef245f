"""The experts' half and the 4-bit weights inside the model and the decoder.

* ``_moe`` over the store's weights against tests/ffn_oracle.py;
* a model with ``weight_format="mx4"`` against a bf16 model over the values its
  codes stand for (exact in bf16): the same layer, its projections summed in
  another order, so within the layers' own bar of 2e-2;
* ``MixDecoder(ffn=True)``: graph replays equal eager launches bit for bit, a step
  equals the layer methods within 2e-2, the captured k-token step equals the eager
  one bit for bit, and k tokens equal k single steps within 2e-2 (where no
  token lies between two experts: the inputs of later layers differ by roundings,
  and the seeds have no such token).
"""

from __future__ import annotations

import os
import sys

import pytest
import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), "golden"))
import inputs as gi  # noqa: E402

import ffn_oracle as fo  # noqa: E402
from margins import record, rel_err  # noqa: E402

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF = torch.bfloat16
N_LAYERS, EXPERTS, TOP_K, INTER, SHARED = 4, 12, 3, 96, 2
BAR = 2e-2


def moe_weights(layer, seed, dtype=BF, hidden=2048):
    r = gi.rng(seed)
    p = f"blk.{layer}.ffn_"
    return {
        p + "gate_inp.weight": gi.normal(r, (EXPERTS, hidden), hidden ** -0.5, dtype),
        p + "gate_exps.weight": gi.normal(r, (EXPERTS, INTER, hidden), hidden ** -0.5, dtype),
        p + "up_exps.weight": gi.normal(r, (EXPERTS, INTER, hidden), hidden ** -0.5, dtype),
        p + "down_exps.weight": gi.normal(r, (EXPERTS, hidden, INTER), INTER ** -0.5, dtype),
        p + "gate_shexp.weight": gi.normal(r, (SHARED * INTER, hidden), hidden ** -0.5, dtype),
        p + "up_shexp.weight": gi.normal(r, (SHARED * INTER, hidden), hidden ** -0.5, dtype),
        p + "down_shexp.weight": gi.normal(r, (hidden, SHARED * INTER), INTER ** -0.5, dtype),
        p + "gate_inp_shexp.weight": gi.normal(r, (1, hidden), hidden ** -0.5, dtype),
    }


def stack_weights():
    w = {}
    for l in range(N_LAYERS):
        w.update(gi.qsa_weights(l, 100 + l, BF) if (l + 1) % 4 == 0 else gi.dn_weights(l, 100 + l, BF))
        w.update(gi.hc_weights(f"blk.{l}.hc_attn", 200 + l, BF))
        w.update(gi.hc_weights(f"blk.{l}.hc_ffn", 300 + l, BF))
        w.update(moe_weights(l, 400 + l))
    return w


PROJECTIONS = ("attn_qkv", "attn_gate", "ssm_beta", "ssm_alpha", "ssm_out", "attn_q", "attn_k", "attn_v", "attn_output",
               "indexer.q_proj", "indexer.k_proj")


def is_quantised(name):
    short = name.split(".", 2)[2]
    return short.removesuffix(".weight") in PROJECTIONS or short.endswith(("exps.weight", "_shexp.weight")) \
        and "gate_inp" not in short


@pytest.fixture(scope="module")
def models(gpu):
    """(package, weights, bf16 model, 4-bit model, bf16 model over the 4-bit values)."""
    qm = gpu
    w = stack_weights()
    cfg = qm.MixConfig(num_experts_per_tok=TOP_K)
    values = {n: (qm.mx4_quantize(t.to(DEV)).dequantize(BF).cpu() if is_quantised(n) else t) for n, t in w.items()}
    # (a shared expert's down projection is quantised per expert: blocks of 32 do not cross its 96 columns)
    make = lambda weights, **kw: qm.Qwen4MixModel(cfg, gi.FakeStore(weights), device=DEV, **kw)  # noqa: E731
    return qm, w, make(w), make(w, weight_format="mx4"), make(values)


def new_cache(qm, model, batch=1):
    cache = qm.MixHybridCache(N_LAYERS, model.config, batch=batch, max_ctx=4096, device=DEV, dtype=BF, page_table="random",
                              seed=3)
    cache.ensure_allocated()
    return cache


def residuals(n, rows=1, k=1, seed=11):
    r = gi.rng(seed)
    return [gi.normal(r, (rows, k, 4 * 2048)).to(BF).to(DEV) for _ in range(n)]


@pytest.mark.parametrize("t", [1, 3, 40])
def test_moe_method_matches_oracle(models, t):
    qm, w, model, _, _ = models
    x = gi.normal(gi.rng(t), (1, t, 2048)).to(BF).to(DEV)
    f = {n.split("ffn_")[1].removesuffix(".weight"): v.to(DEV).double() for n, v in w.items() if n.startswith("blk.1.ffn_")}
    shared = (f["gate_shexp"].view(SHARED, INTER, -1), f["up_shexp"].view(SHARED, INTER, -1),
              f["down_shexp"].view(-1, SHARED, INTER).transpose(0, 1))
    want, bound = fo.moe(x[0], f["gate_inp"], f["gate_exps"], f["up_exps"], f["down_exps"], TOP_K, shared=shared,
                         shared_router=f["gate_inp_shexp"][0])
    got = model._moe(x, 1)
    assert got.shape == x.shape
    assert record("bound", fo.within(got[0], want, bound, BF), 1.0) <= 1.0


@pytest.mark.parametrize("seq", [1, 5, 70, 200])
def test_mx4_layers_match_their_values(models, seq):
    qm, _, _, packed, values = models
    x = gi.hidden_states(seq, seq, BF).to(DEV)
    for layer in (0, 3):
        outs = []
        for m in (packed, values):
            c = new_cache(qm, m)
            if layer == 3:
                outs.append((m._full_attention(x, 3, None, None, c, 0), m._indexer_mask(x, 3, None, None, new_cache(qm, m), seq, 0)))
            else:
                outs.append((m._linear_attention(x, 0, c), None))
        assert rel_err(outs[0][0], outs[1][0], BAR) < BAR
        if layer == 3:
            assert torch.equal(outs[0][1], outs[1][1])            # below the budget: exactly causal
    ids = [qm.moe_route(x, m.moe_weights(2, BF).router, TOP_K)[0] for m in (packed, values)]
    assert torch.equal(*ids)
    assert rel_err(packed._moe(x, 2), values._moe(x, 2), BAR) < BAR


@pytest.mark.parametrize("fmt", ["act", "mx4"])
def test_decoder_steps_with_experts(models, fmt):
    qm, _, plain, packed, _ = models
    model = plain if fmt == "act" else packed
    xs = residuals(5)
    eager_cache = new_cache(qm, model)
    dec = qm.MixDecoder(model, eager_cache, ffn=True)
    eager = [dec.step_eager(x).clone() for x in xs]
    cache = new_cache(qm, model)
    dec = qm.MixDecoder(model, cache, ffn=True)
    junk = torch.randn(256, 256, device=DEV)
    for x, want in zip(xs, eager):
        out = dec.step(x)
        torch.cuda.synchronize()
        junk = torch.tanh(junk @ junk.t() * 1e-3)
        assert torch.equal(out, want)
    # the layer methods, one token at a time
    cache = new_cache(qm, model)
    for i, x in enumerate(xs):
        h = x
        for l in range(N_LAYERS):
            mixed, _, inject = model._gated_residual(h, l, "attn")
            branch = (model._full_attention(mixed, l, None, None, cache, i) if model.config.is_full_attention(l)
                      else model._linear_attention(mixed, l, cache))
            h = model._reinject(h, branch, inject)
            mixed, _, inject = model._gated_residual(h, l, "ffn")
            h = model._reinject(h, model._moe(mixed, l), inject)
        assert rel_err(eager[i], h, BAR) < BAR
    # without the experts a step is what it was
    cache = new_cache(qm, model)
    dec = qm.MixDecoder(model, cache)
    assert not torch.equal(dec.step(xs[0]), eager[0])


@pytest.mark.parametrize("fmt", ["act", "mx4"])
@pytest.mark.parametrize("k", [2, 5, 20])
def test_verify_step_with_experts(models, fmt, k):
    qm, _, plain, packed, _ = models
    model = plain if fmt == "act" else packed
    rows = residuals(1, k=k, seed=40 + k)[0]
    eager = qm.MixDecoder(model, new_cache(qm, model), ffn=True).step_n(rows).clone()
    dec = qm.MixDecoder(model, new_cache(qm, model), ffn=True)
    snap = dec.snapshot()
    for _ in range(3):
        dec.restore(snap)
        got = dec.step_n_graph(rows).clone()
        torch.cuda.synchronize()
        assert torch.equal(got, eager)
    single = qm.MixDecoder(model, new_cache(qm, model), ffn=True)
    steps = torch.cat([single.step(rows[:, i:i + 1]).clone() for i in range(k)], 1)
    assert rel_err(eager, steps, BAR) < BAR


def test_batched_step_equals_single_rows(models):
    """Rows of a batch pass the experts as single rows do (the same experts, sums
    in another order)."""
    qm, _, model, _, _ = models
    x = residuals(1, rows=3, seed=70)[0]
    both = qm.MixDecoder(model, new_cache(qm, model, 3), ffn=True).step(x).clone()
    for b in range(3):
        one = qm.MixDecoder(model, new_cache(qm, model), ffn=True).step(x[b:b + 1])
        assert rel_err(both[b:b + 1], one, BAR) < BAR


def test_weight_format_is_checked(models):
    qm, w, _, _, _ = models
    with pytest.raises(ValueError, match="weight_format"):
        qm.Qwen4MixModel(qm.MixConfig(), gi.FakeStore(w), device=DEV, weight_format="int4")
    bad = dict(w)
    bad["blk.0.ffn_gate_shexp.weight"] = bad["blk.0.ffn_gate_shexp.weight"][:100]
    m = qm.Qwen4MixModel(qm.MixConfig(num_experts_per_tok=TOP_K), gi.FakeStore(bad), device=DEV)
    with pytest.raises(ValueError, match="multiple"):
        m._moe(torch.zeros(1, 1, 2048, dtype=BF, device=DEV), 0)
