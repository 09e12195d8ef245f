"""The experts' and the 4-bit weights' entry points in states that a program around
them brings about: buffers used again, transforms of autograd, tracing, magnitudes
beyond float's range, very wide weights, skewed routers."""

from __future__ import annotations

import copy
import threading

import pytest
import torch
import torch.autograd.forward_ad as fw
from torch.fx.experimental.proxy_tensor import make_fx

import ffn_oracle as fo
from margins import record

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16, F32 = torch.bfloat16, torch.float32


def normal(seed, *shape, dtype=F32, scale=1.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return (torch.randn(*shape, generator=g, device=DEV) * scale).to(dtype)


def layer_tensors(seed, e, h, i, shared, dtype):
    """(router, [gate, up, down], shared (gate, up, down), shared_router)"""
    def mats(s, n):
        return [normal(s, n, i, h, dtype=dtype, scale=h ** -0.5), normal(s + 1, n, i, h, dtype=dtype, scale=h ** -0.5),
                normal(s + 2, n, h, i, dtype=dtype, scale=i ** -0.5)]
    return (normal(seed, e, h, dtype=dtype, scale=h ** -0.5), mats(seed + 1, e), mats(seed + 4, shared),
            normal(seed + 7, h, dtype=dtype, scale=h ** -0.5))


@pytest.mark.parametrize("fmt", ["plain", "mx4"])
@pytest.mark.parametrize("t", [1, 5, 40])
def test_a_layer_keeps_its_weights_when_their_buffers_are_used_again(gpu, fmt, t):
    router, mats, shared, shared_router = layer_tensors(1, 8, 96, 64, 1, BF16)
    lay = gpu.mx4_quantize if fmt == "mx4" else (lambda m: m)
    w = gpu.MoeWeights(router, *(lay(m) for m in mats), top_k=2, shared=[lay(m) for m in shared], shared_router=shared_router)
    x = normal(t, t, 96, dtype=BF16)
    want = gpu.moe(x, w)
    for buf in (router, shared_router, *mats, *shared):
        buf.copy_(normal(99, *buf.shape, dtype=BF16))              # the next layer's
        assert torch.equal(gpu.moe(x, w), want)


@pytest.mark.parametrize("fmt", ["act", "mx4"])
def test_a_model_keeps_a_layers_router_when_the_store_changes(gpu, fmt):
    """A store whose tensors are on the device already, in the activations' type."""
    router, (gate, up, down), (sg, su, sd), row = layer_tensors(5, 8, 96, 64, 1, BF16)
    blk = {"gate_inp": router, "gate_exps": gate, "up_exps": up, "down_exps": down, "gate_shexp": sg[0], "up_shexp": su[0],
           "down_shexp": sd[0], "gate_inp_shexp": row.view(1, -1)}

    class Store:
        def get(self, name):
            return blk[name.split("ffn_")[1].removesuffix(".weight")]

    model = gpu.Qwen4MixModel(gpu.MixConfig(hidden_size=96, num_experts_per_tok=2), Store(), device=DEV, weight_format=fmt)
    x = normal(2, 1, 7, 96, dtype=BF16)
    want = model._moe(x, 0)
    for t in blk.values():
        t.neg_()
    assert torch.equal(model._moe(x, 0), want)


@pytest.mark.parametrize("dtype,t,e", [(BF16, 2000, 64), (F32, 2600, 160)])
def test_shared_gate_beyond_floats_range(gpu, dtype, t, e):
    """Products of the shared experts' row past float's range that cancel: with many
    rows (the matrix cores' sums) as with one."""
    h, i = 1024, 32
    router, mats, shared, row = layer_tensors(11, e, h, i, 1, dtype)
    row[0], row[1] = 2.0 ** 120, -2.0 ** 120
    x = normal(12, t, h, dtype=dtype)
    x[3] = 0
    x[3, :2] = 2.0 ** 30                                            # 2^150 - 2^150: the gate is 1/2
    x[t - 1] = 0
    x[t - 1, 0] = x[t - 1, 1] = -2.0 ** 10
    x[7, :2] = 0
    w = gpu.MoeWeights(router, *mats, top_k=2, shared=shared, shared_router=row)
    got = gpu.moe(x, w)
    pick = [0, 3, 7, 8, t - 1]
    want, bound = fo.moe(x[pick], router.double(), *(m.double() for m in mats), 2, shared=[m.double() for m in shared],
                         shared_router=row)
    assert record("bound", fo.within(got[pick], want, bound, dtype), 1.0) <= 1.0
    for r in pick:
        assert record("alone", fo.within(gpu.moe(x[r:r + 1], w)[0], want[pick.index(r)], bound[pick.index(r)], dtype), 1.0) <= 1.0


def calls(qm, seed=21):
    """(name, call on x [rows, 96] bf16) of every operator that takes activations."""
    router, mats, shared, row = layer_tensors(seed, 8, 96, 64, 1, BF16)
    q = qm.mx4_quantize(mats[0][0])
    w = qm.MoeWeights(router, *mats, top_k=2, shared=shared, shared_router=row)
    return [("linear", lambda x: qm.mx4_linear(x, q)), ("sections", lambda x: qm.mx4_linear(x, q, sections=[60, 4])[1]),
            ("route", lambda x: qm.moe_route(x, router, 2)[1]), ("moe", lambda x: qm.moe(x, w)),
            ("quantize", lambda x: qm.mx4_quantize(x).dequantize())]


@pytest.mark.filterwarnings("ignore")
@pytest.mark.parametrize("t", [1, 20])
def test_derivatives_and_traces_are_refused(gpu, t):
    x = normal(t, t, 96, dtype=BF16)
    for name, call in calls(gpu):
        want = call(x)
        with fw.dual_level():
            with pytest.raises(RuntimeError, match="tangent"):
                call(fw.make_dual(x, torch.ones_like(x)))
            assert torch.equal(call(x), want), name
        with pytest.raises(RuntimeError, match="traced"):
            torch.jit.trace(call, x)
        with pytest.raises(RuntimeError, match="traced"):
            make_fx(call)(x)
        for f in (lambda v: torch.func.jvp(call, (v,), (v,)), torch.func.grad(lambda v: call(v).float().sum()),
                  lambda v: torch.vmap(call)(v[None])):
            with pytest.raises(RuntimeError):
                f(x)
        assert torch.equal(call(x), want), name


@pytest.mark.filterwarnings("ignore")
def test_calls_inside_a_compiled_function(gpu):
    x = normal(3, 20, 96, dtype=BF16)
    for name, call in calls(gpu):
        compiled = torch.compile(lambda v: call(v * 2) + 1, backend="eager")
        for _ in range(2):
            assert torch.equal(compiled(x), call(x * 2) + 1), name


@pytest.mark.parametrize("fmt", ["plain", "mx4"])
def test_a_layer_does_not_change_once_made(gpu, fmt):
    """What a call of some row count keeps holds for every other: nothing of it can be
    replaced."""
    router, mats, shared, row = layer_tensors(31, 8, 96, 64, 1, BF16)
    lay = gpu.mx4_quantize if fmt == "mx4" else (lambda m: m)
    w = gpu.MoeWeights(router, *(lay(m) for m in mats), top_k=2, shared=[lay(m) for m in shared], shared_router=row)
    x = normal(32, 40, 96, dtype=BF16)
    want = gpu.moe(x, w)
    for name, value in (("top_k", 3), ("normalize", False), ("router", router), ("down", w.up), ("shared", 0),
                        ("shared_router", None), ("s_down", None), ("hidden", 64), ("ptrs", None)):
        with pytest.raises(AttributeError, match="does not change"):
            setattr(w, name, value)
    for part in (w.gate, w.down, w.s_up):
        with pytest.raises(AttributeError, match="does not change"):
            part.data = part.data.clone()
    assert torch.equal(gpu.moe(x, w), want)
    other = copy.copy(w)                                            # a shallow copy shares the memory
    assert torch.equal(gpu.moe(x, other), want) and other.down.data.data_ptr() == w.down.data.data_ptr()


# Few rows of weights so wide that they alone make more workgroups than the chip holds:
# both sides of each border of the choice of kernel (8 | 9, 16 | 17 and 32 | 33 rows), and
# of the widths where it begins (bf16 32768 and 196608 rows of weights, float 131072).
@pytest.mark.parametrize("dtype,n", [(BF16, 32700), (BF16, 33001), (BF16, 196700), (F32, 130900), (F32, 131100)])
@pytest.mark.parametrize("m", [1, 8, 9, 16, 17, 32, 33])
def test_few_rows_of_a_wide_weight(gpu, dtype, n, m):
    k = 160
    q = gpu.mx4_quantize(normal(n, n, k, dtype=dtype, scale=k ** -0.5))
    x = normal(m, m, k, dtype=dtype)
    want, bound = fo.linear(x, q.dequantize(F32))
    got = gpu.mx4_linear(x, q)
    assert record("bound", fo.within(got, want, bound, dtype), 1.0) <= 1.0
    parts = gpu.mx4_linear(x, q, sections=[n - 1000, 999, 1])
    assert torch.equal(torch.cat(parts, -1), got)


# Both sides of the products up to which every logit is summed in double. A weight is
# within 2^-18 of the softmax of those sums (an exponential of a difference below 16
# rounded to float, a float sum, a division), and by 4 B more where the matrix cores
# sum 128 products at a time: B = (129 2^-23) |x| |R[e]| bounds their error.
@pytest.mark.parametrize("dtype,t,e,h", [(BF16, 755, 64, 2048), (BF16, 770, 64, 2048), (F32, 2800, 64, 2048),
                                         (F32, 2850, 64, 2048)])
def test_route_at_the_border_of_its_sums(gpu, dtype, t, e, h):
    x, r = normal(t, t, h, dtype=dtype), normal(h, e, h, dtype=dtype, scale=h ** -0.5)
    ids, w = gpu.moe_route(x, r, 6)
    want_ids, want_w = fo.route(x, r, 6)
    assert torch.equal(ids, want_ids)
    lim = 2.0 ** -18 + 4 * 129 * 2.0 ** -23 * x.double().norm(dim=-1) * r.double().norm(dim=-1).max()
    assert record("bound", ((w.double() - want_w).abs() / want_w / lim[:, None]).max().item(), 1.0) <= 1.0


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_read_back_of_every_code_and_scale(gpu, dtype):
    """All 16 codes under all 256 scales: subnormal values are exact, those past the
    type's range infinite, scale 255 NaN."""
    codes = torch.arange(16, dtype=torch.uint8, device=DEV)
    codes = (codes | codes.flip(0) << 4).repeat(256, 1)
    scales = torch.arange(256, dtype=torch.uint8, device=DEV)[:, None]
    q = gpu.Mx4Weight.from_codes(codes, scales)
    got, want = q.dequantize(dtype), fo.mx4_decode(codes, scales)
    assert torch.equal(got[:255].double(), want[:255].to(dtype).double())
    assert torch.equal(torch.signbit(got[:255]), torch.signbit(want[:255])) and bool(got[255].isnan().all())
    tiny = want[0].abs()[want[0] != 0].min().item()
    assert tiny == 2.0 ** -128 and got[0].double().abs()[got[0] != 0].min().item() == tiny
    back = q.plain()
    assert torch.equal(back[0], codes) and torch.equal(back[1], scales)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("m,n", [(2, 70), (9, 70), (40, 300), (60, 4090), (170, 4090), (300, 4090), (700, 4090),
                                 (2000, 1000), (5, 33000), (20, 33000)])
def test_an_infinite_activation_reaches_every_output(gpu, dtype, m, n):
    """inf times a weight is that infinity, inf times zero is NaN: no output of the row
    stays finite, whichever kernel has it."""
    k = 224
    w = normal(n, n, k, dtype=dtype)
    w[::7, k - 1] = 0
    q = gpu.mx4_quantize(w)
    column = q.dequantize(F32)[:, k - 1]
    assert bool((column == 0).any()) and bool((column > 0).any()) and bool((column < 0).any())
    x = normal(m, m, k, dtype=dtype)
    clean = gpu.mx4_linear(x, q)
    x[0, k - 1], x[m - 1, k - 1] = float("inf"), float("-inf")
    got = gpu.mx4_linear(x, q)
    for row, sign in ((0, 1.0), (m - 1, -1.0)):
        assert not bool(got[row].isfinite().any())
        assert torch.equal(got[row].isnan(), column == 0)
        hit = column != 0
        assert torch.equal(torch.sign(got[row].float())[hit], sign * torch.sign(column)[hit])
    assert torch.equal(got[1:m - 1], clean[1:m - 1])


def make(qm, tensors, fmt, top_k, normalize=True):
    """(MoeWeights, the oracle's arguments) of layer_tensors."""
    router, mats, shared, row = tensors
    shared = shared if shared[0].shape[0] else None
    if fmt == "mx4":
        mats, shared = [qm.mx4_quantize(m) for m in mats], None if shared is None else [qm.mx4_quantize(m) for m in shared]
        value = lambda m: m.dequantize().double()  # noqa: E731
    else:
        value = lambda m: m.double()  # noqa: E731
    row = None if shared is None else row
    w = qm.MoeWeights(router, *mats, top_k=top_k, shared=shared, shared_router=row, normalize=normalize)
    return w, dict(zip(("gate", "up", "down"), map(value, mats)), router=router, top_k=top_k, normalize=normalize,
                   shared=None if shared is None else [value(m) for m in shared], shared_router=row)


def check(got, x, args):
    want, bound = fo.moe(x, **args)
    assert got.shape == x.shape and got.dtype == x.dtype
    assert record("bound", fo.within(got, want, bound, x.dtype), 1.0) <= 1.0


# float layers at the borders between the kernels: 16 and 17 tokens; lists by the choosing
# waves and apart, over several rounds of choices; weights read once and more often; logits
# by matrix cores; then layers of many experts, of either type
@pytest.mark.parametrize("fmt", ["plain", "mx4"])
@pytest.mark.parametrize("dtype,t,e,k,h,i,shared", [
    (F32, 16, 24, 4, 288, 160, 1), (F32, 17, 24, 4, 288, 160, 1), (F32, 300, 8, 2, 160, 96, 1), (F32, 90, 16, 2, 160, 96, 0),
    (F32, 3000, 32, 6, 64, 32, 0), (F32, 6000, 60, 4, 1056, 32, 1), (F32, 40, 1024, 32, 32, 32, 0), (F32, 3, 32, 32, 64, 32, 32),
    (BF16, 1, 256, 8, 512, 128, 1), (BF16, 50, 512, 10, 256, 64, 1), (BF16, 400, 256, 8, 256, 64, 0),
    (F32, 12, 300, 6, 128, 64, 1), (BF16, 2000, 640, 4, 128, 32, 0)])
def test_float_layers_and_many_experts(gpu, fmt, dtype, t, e, k, h, i, shared):
    print(f"moe {dtype} {fmt} t={t} e={e} k={k} h={h} i={i} shared={shared}", flush=True)
    w, args = make(gpu, layer_tensors(t + e, e, h, i, shared, dtype), fmt, k, normalize=t % 2 == 0)
    x = normal(t, t, h, dtype=dtype)
    check(gpu.moe(x, w), x, args)


@pytest.mark.parametrize("fmt", ["plain", "mx4"])
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("t,e,k", [(6, 64, 6), (16, 256, 8), (150, 64, 6), (900, 160, 4)])
def test_skewed_routers(gpu, fmt, dtype, t, e, k):
    """Load as trained routers have it: the tokens share a direction, and the experts'
    rows follow it by falling amounts, so a few experts take most rows, most none."""
    h, i = 160, 64
    tensors = layer_tensors(41, e, h, i, 1, dtype)
    shared_direction = normal(42, h)
    order = torch.randperm(e, generator=torch.Generator().manual_seed(43)).to(DEV)
    lean = 4.0 / (1.0 + order.float())
    tensors[0].copy_(tensors[0] + (lean[:, None] * shared_direction * h ** -0.5).to(dtype))
    x = normal(t, t, h, dtype=dtype) + shared_direction.to(dtype)
    w, args = make(gpu, tensors, fmt, k)
    ids = gpu.moe_route(x, tensors[0], k)[0]
    counts = torch.bincount(ids.flatten().long(), minlength=e)
    assert counts.max().item() > 0.8 * t
    check(gpu.moe(x, w), x, args)


def test_the_largest_calls(gpu):
    """As many rows as one call takes, and one more."""
    h, t = 32, 262140
    w, args = make(gpu, layer_tensors(51, 4, h, 32, 0, BF16), "plain", 1)
    x = normal(52, t + 1, h, dtype=BF16)
    got = gpu.moe(x[:t], w)
    want, bound = fo.moe(x[:t], **args)
    assert record("bound", fo.within(got, want, bound, BF16), 1.0) <= 1.0
    for call in (lambda: gpu.moe(x, w), lambda: gpu.moe_route(x, args["router"], 1)):
        with pytest.raises(gpu.native.QmError, match="262140"):
            call()
    del got, want, bound
    m = 16 * 65535
    for dtype in (BF16, F32):
        q = gpu.mx4_quantize(normal(53, 20, h, dtype=dtype))
        x = normal(54, m + 1, h, dtype=dtype)
        want, bound = fo.linear(x[:m], q.dequantize(F32))
        assert record("bound", fo.within(gpu.mx4_linear(x[:m], q), want, bound, dtype), 1.0) <= 1.0
        with pytest.raises(gpu.native.QmError, match="1048560"):
            gpu.mx4_linear(x, q)


@pytest.mark.parametrize("fmt", ["plain", "mx4"])
def test_calls_from_threads(gpu, fmt):
    """Host threads with a stream each, every thread's first calls among them."""
    e, h, i = 16, 256, 64
    w, args = make(gpu, layer_tensors(61, e, h, i, 1, BF16), fmt, 4)
    q = gpu.mx4_quantize(normal(62, 4000, h, dtype=BF16))
    sizes = (1, 12, 90, 700)
    xs = [[normal(70 + n, t, h, dtype=BF16) for t in sizes] for n in range(4)]
    got = [None] * len(xs)

    def work(n):
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            got[n] = [(gpu.moe(x, w), gpu.mx4_linear(x, q), *gpu.moe_route(x, args["router"], 4)) for _ in range(5) for x in xs[n]]
        stream.synchronize()

    torch.cuda.synchronize()
    threads = [threading.Thread(target=work, args=(n,)) for n in range(len(xs))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for n, seq in enumerate(xs):
        want = [(gpu.moe(x, w), gpu.mx4_linear(x, q), *gpu.moe_route(x, args["router"], 4)) for x in seq]
        assert all(torch.equal(a, b) for rep in range(5) for one, ref in zip(got[n][rep * len(seq):], want)
                   for a, b in zip(one, ref))
