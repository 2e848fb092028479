"""Layers of a GGUF file as 8-bit integers: loading, products, the MoE layer from its logits on, and the C-ABI under all of it."""
import numpy as np
import pytest
import torch

from gguf_b200 import capi, synth
from test_int8_ops import TINY, check_product, codes_of, experts, moe_want

DEV = "cuda"


def blocks(t, n, k, seed=0):
    return torch.from_numpy(synth.make_weight(t, n, k, seed=seed)).to(DEV)


def linear(types, rows, k, dtype=torch.float16):
    from vllm_gguf_plugin.quantization import Int8LinearMethod

    method, layer = Int8LinearMethod(None), torch.nn.Module()
    method.create_weights(layer, k, rows, k, sum(rows), dtype)
    parts = [blocks(t, r, k, seed=i) for i, (t, r) in enumerate(zip(types, rows))]
    for sid, t, w in zip([None] if len(rows) == 1 else "qkv", types, parts):
        layer.weight.weight_loader(layer.weight, w, sid)
        layer.weight_type.weight_loader(layer.weight_type, torch.tensor(t), sid)
    method.process_weights_after_loading(layer)
    values = torch.cat([capi.dequantize(w, t, w.shape[0], k, torch.float32) for t, w in zip(types, parts)])
    return method, layer, values


@pytest.mark.gpu
@pytest.mark.parametrize("types,rows,k", [((8,), [300], 544), ((12,), [1024], 2048), ((16,), [128], 256), ((12, 12, 14), [512, 128, 128], 768), ((2,), [64], 96)])
@pytest.mark.parametrize("m", [1, 5, 70])
def test_linear_layer(native_libs, types, rows, k, m):
    method, layer, values = linear(types, rows, k)
    w, ws = codes_of(values)
    assert torch.equal(layer.int8_weight.double(), w) and layer.weight.numel() == 0
    assert bool(((layer.int8_scales.double() - ws).abs() <= 2.0 ** -24 * ws).all())
    for dtype in (torch.float16, torch.bfloat16, torch.float32):
        x = torch.randn(m, k, device=DEV).to(dtype)
        bias = torch.randn(sum(rows), device=DEV, dtype=torch.float32)
        check_product(method.apply(layer, x), *codes_of(x), w, layer.int8_scales, None, dtype)
        check_product(method.apply(layer, x, bias), *codes_of(x), w, layer.int8_scales, bias.to(dtype), dtype)
    kept = layer.int8_weight.data_ptr()
    method.process_weights_after_loading(layer)   # nothing new: nothing happens
    assert layer.int8_weight.data_ptr() == kept


@pytest.mark.gpu
def test_linear_layer_against_its_blocks(native_libs):
    """Row scales instead of block scales, token scales instead of one for 32 values: two roundings of at most half a code of the row's 127, as
    independent errors (a sum of K products of them, root mean squares): far below 2 % of the product for normal data."""
    from vllm_gguf_plugin.quantization import GGUFLinearMethod

    method, layer, values = linear((8,), [512], 2048)
    x = torch.randn(40, 2048, device=DEV)
    want = x.double() @ values.double().T
    got = method.apply(layer, x).double()
    assert float((got - want).norm() / want.norm()) < 0.02
    assert issubclass(type(method), GGUFLinearMethod)


@pytest.mark.gpu
def test_reloading_and_first_product_behind_it(native_libs):
    from vllm_gguf_plugin.quantization import Int8LinearMethod

    files = [blocks(8, 4096, 1024, seed=s) for s in (1, 2)]
    x = torch.randn(1, 1024, device=DEV).half()
    want = []
    for w in files:
        codes, scales = capi.int8_quantize(capi.dequantize(w, 8, 4096, 1024, torch.float32))
        torch.cuda.synchronize()
        want.append(capi.int8_mul_mat(codes, scales, x))
    method, layer = Int8LinearMethod(None), torch.nn.Module()
    method.create_weights(layer, 1024, [4096], 1024, 4096, torch.float16)
    got = []
    for i in range(20):
        layer.weight.weight_loader(layer.weight, files[i & 1].clone(), None)
        layer.weight_type.weight_loader(layer.weight_type, torch.tensor(8), None)
        method.process_weights_after_loading(layer)
        got.append(method.apply(layer, x))
    torch.cuda.synchronize()
    assert all(torch.equal(y, want[i & 1]) for i, y in enumerate(got))


def moe_layer(method, t13, t2, e, h, i):
    layer = torch.nn.Module()
    method.create_weights(layer, e, h, i, torch.float16)
    w1, w3, w2 = (np.stack([synth.make_weight(t, n, k, seed=100 * s + j) for j in range(e)]) for s, t, n, k in ((1, t13, i, h), (3, t13, i, h), (2, t2, h, i)))
    for sid, w, name, t in (("w1", w1, "w13", t13), ("w3", w3, "w13", t13), ("w2", w2, "w2", t2)):
        param, kind = getattr(layer, name + "_weight"), getattr(layer, name + "_weight_type")
        param.weight_loader(param, torch.from_numpy(w).to(DEV), "experts", shard_id=sid, expert_id=0)
        kind.weight_loader(kind, torch.tensor(t), "experts", shard_id=sid)
    return layer


@pytest.mark.gpu
@pytest.mark.parametrize("tokens", [1, 9, 150])
def test_moe_layer_from_its_logits(native_libs, tokens):
    """Gate, route, experts and sum, as a model runs them, on blocks and on 8-bit integers."""
    from vllm_gguf_plugin import ops
    from vllm_gguf_plugin.quantization import GGUFMoEMethod, Int8MoEMethod, int8_rows

    e, h, i = 16, 512, 256
    gguf, int8 = GGUFMoEMethod(None), Int8MoEMethod(None)
    layer = moe_layer(gguf, 8, 8, e, h, i)
    w13 = int8_rows(layer.w13_weight.data.reshape(e * 2 * i, -1), 8)
    w2 = int8_rows(layer.w2_weight.data.reshape(e * h, -1), 8)
    layer8 = moe_layer(int8, 8, 8, e, h, i)
    int8.process_weights_after_loading(layer8)
    int8.process_weights_after_loading(layer8)
    assert torch.equal(layer8.w13_int8.reshape(e * 2 * i, h), w13[0]) and torch.equal(layer8.w2_scales.flatten(), w2[1]) and layer8.w2_weight.numel() == 0
    for l in (layer, layer8):
        l.top_k, l.scoring_func, l.use_grouped_topk, l.num_expert_group, l.topk_group, l.routed_scaling_factor = 4, "sigmoid", True, 4, 2, 1.5
        l.e_score_correction_bias = torch.linspace(-0.1, 0.1, e, device=DEV)
    gen = torch.Generator(device=DEV).manual_seed(tokens)
    x = (torch.randn(tokens, h, device=DEV, generator=gen) * 0.1).half()
    logits = (x.float() @ torch.randn(h, e, device=DEV, generator=gen))
    weights_, ids = ops.moe_route(logits, 4, scoring="sigmoid", bias=layer.e_score_correction_bias, n_group=4, topk_group=2, scale=1.5)
    got = gguf.route(layer, logits)
    assert torch.equal(got[0], weights_) and torch.equal(got[1], ids)
    y = int8.apply_logits(layer8, x, logits)
    want, room = moe_want(x, layer8.w13_int8, layer8.w13_scales, layer8.w2_int8, layer8.w2_scales, weights_, ids, "silu")
    room = room + 2.0 ** -11 * (want.abs() + room) + TINY[torch.float16] + 2.0 ** -22 * want.abs()
    assert bool(((y.double() - want).abs() <= room).all())
    blocks_y = gguf.apply_logits(layer, x, logits)
    assert torch.equal(blocks_y, gguf.apply(layer, x, weights_, ids))
    # the same layer on blocks and on rows: two more roundings of half a code of 127 in each of two products
    assert float((y.double() - blocks_y.double()).norm() / blocks_y.double().norm()) < 0.05
    layer8.activation = "relu"
    with pytest.raises(NotImplementedError):
        int8.apply(layer8, x, weights_, ids)


@pytest.mark.gpu
def test_layer_of_more_than_256_experts_behind_the_router(native_libs):
    """Block formats, a padded row and a row with fewer experts than places: nothing comes from the places that are left."""
    from vllm_gguf_plugin.quantization import GGUFMoEMethod

    e, h, i = 260, 64, 32
    method = GGUFMoEMethod(None)
    layer = moe_layer(method, 8, 8, e, h, i)
    layer.top_k = 4
    gen = torch.Generator(device=DEV).manual_seed(3)
    x = torch.randn(6, h, device=DEV, generator=gen).half()
    logits = torch.randn(6, e, device=DEV, generator=gen)
    logits[2] = float("-inf")
    logits[4] = float("-inf")
    logits[4, 259] = 1.0
    junk = torch.full((1 << 20,), float("nan"), device=DEV)   # (what the next buffers find)
    del junk
    y = method.apply_logits(layer, x, logits)
    weights_, ids = method.route(layer, logits)
    assert ids[2].tolist() == [-1] * 4 and ids[4].tolist() == [259, -1, -1, -1]
    assert not bool(y[2].any()) and bool(torch.isfinite(y).all())
    alone = method.apply(layer, x[4:5], torch.ones(1, 1, device=DEV), torch.full((1, 1), 259, dtype=torch.int32, device=DEV))
    assert torch.equal(y[4:5], alone)


@pytest.mark.gpu
def test_moe_layer_loaded_again_in_part(native_libs):
    """What arrives after the first loading takes the place of what it is, and of nothing else: one projection, one half of one, one expert."""
    from vllm_gguf_plugin.quantization import Int8MoEMethod, int8_rows

    e, h, i, t = 4, 96, 64, 8
    method = Int8MoEMethod(None)
    layer = moe_layer(method, t, t, e, h, i)
    method.process_weights_after_loading(layer)
    ids, weights_ = torch.tensor([[0, 1], [2, 3], [3, 0]], dtype=torch.int32, device=DEV), torch.full((3, 2), 0.5, device=DEV)
    x = torch.randn(3, h, device=DEV, generator=torch.Generator(device=DEV).manual_seed(1)).half()

    def state():
        return [layer.w13_int8.clone(), layer.w13_scales.clone(), layer.w2_int8.clone(), layer.w2_scales.clone()]

    def load(name, sid, w, expert=0):
        param = getattr(layer, name + "_weight")
        param.weight_loader(param, w, "experts", shard_id=sid, expert_id=expert)

    def rows(w):
        codes, scales = int8_rows(w.reshape(-1, w.shape[-1]), t)
        return codes.unflatten(0, w.shape[:-1]), scales.view(w.shape[:-1])

    want, n = state(), 0
    for name, sid, at, lead, r0, k in (("w2", "w2", 2, (e, h), 0, i), ("w13", "w3", 0, (e, i), i, h), ("w13", "w1", 0, (i,), 0, h), ("w2", "w2", 2, (h,), 0, i)):
        n += 1
        w = blocks(t, int(np.prod(lead)), k, seed=1000 + n).unflatten(0, lead)
        load(name, sid, w, expert=3)
        method.process_weights_after_loading(layer)
        part = slice(None) if len(lead) == 2 else 3
        want[at][part, r0:r0 + lead[-1]], want[at + 1][part, r0:r0 + lead[-1]] = rows(w)
        assert all(torch.equal(a, b) for a, b in zip(state(), want)), (name, sid)
        y = method.apply(layer, x, weights_, ids)
        fresh = torch.nn.Module()
        fresh.w13_int8, fresh.w13_scales, fresh.w2_int8, fresh.w2_scales = layer.w13_int8, want[1], layer.w2_int8, want[3]
        assert torch.equal(y, method.apply(fresh, x, weights_, ids))
    # all of it again, an expert at a time
    for j in range(e):
        for name, sid, r, k in (("w13", "w1", i, h), ("w13", "w3", i, h), ("w2", "w2", h, i)):
            load(name, sid, blocks(t, r, k, seed=50 * j + r + len(sid)), expert=j)
    whole = {n_: getattr(layer, n_ + "_weight").data.clone() for n_ in ("w13", "w2")}
    method.process_weights_after_loading(layer)
    got = state()
    for at, n_ in ((0, "w13"), (2, "w2")):
        codes, scales = rows(whole[n_])
        assert torch.equal(got[at], codes) and torch.equal(got[at + 1], scales)


def test_route_reads_the_layer(monkeypatch, native_libs):
    from vllm_gguf_plugin import ops
    from vllm_gguf_plugin.quantization import GGUFMoEMethod

    seen = {}
    monkeypatch.setattr(ops, "moe_route", lambda logits, top_k, **kw: seen.update(kw, top_k=top_k))
    layer = torch.nn.Module()
    layer.top_k = 3
    GGUFMoEMethod.route(layer, None)
    assert seen == dict(top_k=3, scoring="softmax", bias=None, n_group=1, topk_group=1, renormalize=True, scale=1.0)
    layer.num_expert_group, layer.topk_group, layer.renormalize, layer.routed_scaling_factor = 8, 4, False, 2.5
    GGUFMoEMethod.route(layer, None)      # (groups only where the layer uses them)
    assert (seen["n_group"], seen["topk_group"], seen["renormalize"], seen["scale"]) == (1, 1, False, 2.5)
    layer.use_grouped_topk = True
    GGUFMoEMethod.route(layer, None)
    assert (seen["n_group"], seen["topk_group"]) == (8, 4)


@pytest.mark.parametrize("name,value", [("custom_routing_function", lambda *a: None), ("enable_eplb", True)])
def test_route_refuses_a_layer_that_routes_otherwise(monkeypatch, native_libs, name, value):
    from vllm_gguf_plugin import ops
    from vllm_gguf_plugin.quantization import GGUFMoEMethod

    calls = []
    monkeypatch.setattr(ops, "moe_route", lambda logits, top_k, **kw: calls.append(kw))
    layer = torch.nn.Module()
    layer.top_k = 3
    setattr(layer, name, value)
    for call in (lambda: GGUFMoEMethod.route(layer, None), lambda: GGUFMoEMethod(None).apply_logits(layer, None, None)):
        with pytest.raises(NotImplementedError, match=name):
            call()
    assert not calls
    setattr(layer, name, None if name == "custom_routing_function" else False)
    GGUFMoEMethod.route(layer, None)
    assert len(calls) == 1


def test_rows_of_an_unknown_type_are_refused(native_libs):
    from vllm_gguf_plugin.quantization import int8_rows

    with pytest.raises(NotImplementedError, match="type: 9"):
        int8_rows(torch.zeros(2, 36, dtype=torch.uint8), 9)


@pytest.mark.gpu
def test_c_abi_gives_what_the_operators_give(native_libs):
    from vllm_gguf_plugin import ops

    gen = torch.Generator(device=DEV).manual_seed(6)
    x = torch.randn(20, 200, device=DEV, generator=gen).half()
    q, s = capi.int8_quantize(x)
    assert all(torch.equal(a, b) for a, b in zip((q, s), ops.int8_quantize(x)))
    w, ws = ops.int8_quantize(torch.randn(64, 200, device=DEV, generator=gen))
    for m in (1, 20):
        for flags in (0, 0x100):
            assert torch.equal(capi.int8_mul_mat(w, ws, x[:m], flags=flags), ops.int8_mul_mat(w, ws, x[:m]))
    logits = torch.randn(20, 8, device=DEV, generator=gen)
    weights_, ids = capi.moe_route(logits, 2)
    assert all(torch.equal(a, b) for a, b in zip((weights_, ids), ops.moe_route(logits, 2)))
    w13, s13, w2, s2 = experts(8, 200, 64, gen)
    assert torch.equal(capi.int8_fused_moe(x, w13, s13, w2, s2, weights_, ids), ops.int8_fused_moe(x, w13, s13, w2, s2, weights_, ids, "silu"))
    assert capi.last_status() == 0


@pytest.mark.gpu
def test_compiled_calls_and_modes_take_the_operators(native_libs):
    from torch.utils._python_dispatch import TorchDispatchMode

    from vllm_gguf_plugin import ops

    seen = []

    class Record(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            seen.append(str(func))
            return func(*args, **(kwargs or {}))

    method, layer, _ = linear((8,), [64], 64)
    gen = torch.Generator(device=DEV).manual_seed(6)
    x = torch.randn(3, 64, device=DEV, generator=gen)
    w13, s13, w2, s2 = experts(8, 64, 64, gen)

    def run(x):
        weights_, ids = ops.moe_route(x[:, :8], 2)
        return ops.int8_fused_moe(method.apply(layer, x), w13, s13, w2, s2, weights_, ids, "gelu"), ops.int8_quantize(x)[0]

    want = run(x)
    with Record():
        got = run(x)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    names = {n.split(".")[1] for n in seen if n.startswith("_C_gguf")}
    assert {"moe_route", "int8_mul_mat", "int8_fused_moe", "int8_quantize"} <= names
    compiled = torch.compile(run, fullgraph=True, backend="aot_eager")
    assert all(torch.equal(a, b) for a, b in zip(compiled(x), want))
