"""The 8-bit integer operators (row quantizer, linear product, routed expert step) against their definitions in 64 bits.

Tolerances.  Codes are those of exact arithmetic and are compared for equality.  A scale is one fp32 division: 2^-24 relative.  A
result is D * (q_scale * w_scale) + bias with D exact: q_scale, the conversion of D, two products and a sum are rounded to fp32
once each, at most 5 * 2^-24 of |D| q_scale w_scale + |bias|, and the result once more to its type: eps / 2 of itself, or half
the smallest subnormal."""
import ctypes

import pytest
import torch

from helpers import ROOT  # noqa: F401  (puts the package on the path)

DTYPES = [torch.float32, torch.float16, torch.bfloat16]
TINY = {torch.float32: 2.0 ** -150, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134}


@pytest.fixture(scope="module")
def ops(native_libs):
    from vllm_gguf_plugin import ops

    return ops


def codes_of(x):
    """(codes, scales) of the definition, float64; rows that are not finite have scale NaN and codes 0."""
    x = x.double()
    a = x.abs().amax(1, keepdim=True)
    ok = torch.isfinite(x).all(1, keepdim=True)
    a = torch.where(ok, a, 1.0)
    q = torch.where(ok, torch.round(torch.where(ok, x, 0.0) * 127 / torch.where(a > 0, a, 1.0)), 0.0)
    return q, torch.where(ok, a / 127, float("nan")).squeeze(1)


def weights(rows, k, gen, spread=36.0):
    buf = torch.full((rows, (k + 15) // 16 * 16), 77, dtype=torch.int8, device="cuda")   # (what lies behind K must not count)
    buf[:, :k] = (torch.randn(rows, k, device="cuda", generator=gen) * spread).round().clamp(-128, 127).to(torch.int8)
    return buf[:, :k], (torch.rand(rows, device="cuda", generator=gen) + 0.5) * 1e-3


def check_product(y, q, qs, w, ws, bias, dtype, msg=""):
    d = q.double() @ w.double().T
    part = d * qs.double()[:, None] * ws.double()
    want = part if bias is None else part + bias.double()
    room = 5 * 2.0 ** -24 * (part.abs() + (0 if bias is None else bias.double().abs()))
    room = room + torch.finfo(dtype).eps / 2 * (want.abs() + room) + TINY[dtype]
    assert y.shape == want.shape and y.dtype == dtype
    off = (y.double() - want).abs() - room
    assert bool((off <= 0).all()), f"{msg}: off by {float((y.double() - want).abs().max())}, {int((off > 0).sum())} of {off.numel()} values"


# ---- row quantizer -------------------------------------------------------------------------------------------


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,k", [(1, 1), (1, 15), (3, 16), (7, 33), (1, 4096), (9, 1000), (130, 2048), (5, 2049), (2, 4100), (3, 16384), (2, 16400),
                                    (2, 40007), (1, 131072), (1500, 64), (41003, 48), (21001, 1040), (10003, 2064), (5003, 4109)])
def test_quantize_matches_exact_codes(ops, dtype, rows, k):
    gen = torch.Generator(device="cuda").manual_seed(rows * 7 + k)
    x = torch.randn(rows, k, device="cuda", generator=gen).to(dtype)
    q, s = ops.int8_quantize(x)
    want, scale = codes_of(x)
    assert q.dtype == torch.int8 and q.shape == (rows, k) and s.shape == (rows,) and q.data_ptr() % 16 == 0 and (rows == 1 or q.stride(0) % 16 == 0)
    assert torch.equal(q.double(), want)
    assert bool(((s.double() - scale).abs() <= 2.0 ** -24 * scale).all())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_quantize_halves_zeros_and_what_is_not_finite(ops, dtype):
    inf, nan = float("inf"), float("nan")
    top = torch.finfo(dtype).max
    tiny = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps   # the smallest subnormal
    rows = [
        [2.0, 1.0, -1.0, 0.0, -2.0] + [0.0] * 12,                        # 63.5 and -63.5 go to 64
        [254.0, 1.0, 3.0, 5.0, -1.0, -3.0, -5.0, 7.0] + [0.0] * 9,       # 0.5, 1.5, 2.5 ... to even
        [0.0, -0.0] + [0.0] * 15,
        [1.0, inf] + [1.0] * 15,
        [1.0, -inf] + [1.0] * 15,
        [nan] + [1.0] * 16,
        [0.0] * 16 + [nan],
        [top, -top, top / 2] + [1.0] * 14,
        [tiny, 0.0, -tiny] + [0.0] * 14,
        [3 * tiny, tiny, -tiny, 2 * tiny] + [0.0] * 13,
        [torch.finfo(dtype).smallest_normal, tiny] + [0.0] * 15,
    ]
    x = torch.tensor(rows, dtype=torch.float64).to(dtype).cuda()
    q, s = ops.int8_quantize(x)
    want, scale = codes_of(x)
    assert torch.equal(q.double(), want)
    assert torch.equal(torch.isnan(s), torch.isnan(scale))
    ok = ~torch.isnan(scale)
    assert bool(((s.double() - scale).abs()[ok] <= 2.0 ** -24 * scale[ok] + 2.0 ** -150).all())   # (or half the smallest fp32 subnormal)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_quantize_every_near_half(ops, dtype):
    """Every value of a binade over the largest of the row, so that all roundings next to halves occur."""
    n = 4096
    for top in (1.0, 1.25, 1.9921875, 1.3359375):
        x = torch.linspace(-top, top, n, dtype=torch.float64).to(dtype).cuda()[None].contiguous()
        x[0, 0] = top
        half = ((torch.arange(-127, 127, dtype=torch.float64) + 0.5) * float(x[0, 0]) / 127).to(dtype).cuda()
        x[0, 1:1 + half.numel()] = half
        q, _ = ops.int8_quantize(x)
        assert torch.equal(q.double(), codes_of(x)[0])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_quantize_strides(ops, dtype):
    gen = torch.Generator(device="cuda").manual_seed(5)
    big = torch.randn(40, 333, device="cuda", generator=gen).to(dtype)
    for x in (big[:, 3:100], big[::3, :64], big[:, :320], big[5:6, 1:290], big[:1].expand(6, -1), torch.empty(0, 48, device="cuda", dtype=dtype)):
        q, _ = ops.int8_quantize(x)
        assert torch.equal(q.double(), codes_of(x)[0] if len(x) else q.double())


# ---- linear product ------------------------------------------------------------------------------------------

SIZES = [(1, 1, 1), (1, 1, 16), (1, 7, 33), (1, 128, 128), (2, 129, 127), (1, 4096, 4096), (2, 1000, 2064), (3, 200, 4096), (5, 300, 1040), (7, 128, 14336),
         (8, 513, 5000), (1, 19072, 6144), (4, 19072, 6160), (9, 130, 4096), (16, 256, 1024), (17, 4000, 512), (27, 384, 8192),
         (33, 300, 2048), (64, 640, 4096), (65, 130, 4100), (128, 1000, 640), (200, 256, 14336), (255, 130, 256), (256, 130, 640), (257, 130, 640),
         (300, 4096, 1536), (513, 257, 384), (1000, 520, 1040), (2049, 2100, 400),
         # shared by two, by four; pairs, odd numbers of 128-row tiles among them
         (3, 2050, 9000), (20, 2100, 14000), (90, 1030, 13000), (520, 4224, 12345), (450, 9000, 2080), (2100, 6000, 1030)]


@pytest.mark.gpu
@pytest.mark.parametrize("m,n,k", SIZES)
@pytest.mark.parametrize("dtype", DTYPES)
def test_linear(ops, dtype, m, n, k):
    gen = torch.Generator(device="cuda").manual_seed(m + n + k)
    w, ws = weights(n, k, gen)
    x = torch.randn(m, k, device="cuda", generator=gen).to(dtype)
    bias = torch.randn(n, device="cuda", generator=gen).to(dtype) if (m + n) % 2 else None
    y = ops.int8_mul_mat(w, ws, x, bias)
    q, qs = codes_of(x)
    check_product(y, q, qs, w, ws, bias, dtype, f"{m}x{n}x{k}")
    # the same in two calls, and again: bit for bit
    codes, scales = ops.int8_quantize(x)
    assert torch.equal(ops.int8_mul_mat_prepared(w, ws, codes, scales, dtype, bias), y)
    assert torch.equal(ops.int8_mul_mat(w, ws, x, bias), y)


@pytest.mark.gpu
def test_linear_largest_sums(ops):
    """128 * 127 * 131071 fills 31 bits: nothing saturates or wraps."""
    k = 131071
    buf = torch.full((130, k + 1), -128, dtype=torch.int8, device="cuda")
    w = buf[:, :k]
    ws = torch.ones(130, device="cuda")
    for m in (1, 20):
        x = torch.full((m, k), -127.0, device="cuda")
        x[0] = 127
        y = ops.int8_mul_mat(w, ws, x)
        want = torch.full((m, 130), 127.0 * 128 * k, dtype=torch.float64, device="cuda")
        want[0] *= -1
        assert bool(((y.double() - want).abs() <= 5 * 2.0 ** -24 * want.abs()).all())
    with pytest.raises(RuntimeError, match="size"):
        ops.int8_mul_mat(torch.zeros(1, 131072, dtype=torch.int8, device="cuda"), ws[:1], torch.zeros(1, 131072, device="cuda"))


@pytest.mark.gpu
@pytest.mark.parametrize("m", [1, 40, 300])
def test_linear_rows_that_are_not_finite_stay_alone(ops, m):
    gen = torch.Generator(device="cuda").manual_seed(m)
    w, ws = weights(200, 256, gen)
    x = torch.randn(m, 256, device="cuda", generator=gen)
    clean = ops.int8_mul_mat(w, ws, x)
    x[0, 3], x[m // 2, 5] = float("nan"), float("-inf")
    y = ops.int8_mul_mat(w, ws, x)
    bad = torch.zeros(m, dtype=torch.bool, device="cuda")
    bad[[0, m // 2]] = True
    assert bool(torch.isnan(y[bad]).all()) and torch.equal(y[~bad], clean[~bad])


@pytest.mark.gpu
def test_linear_empty_strided_and_misaligned(ops):
    gen = torch.Generator(device="cuda").manual_seed(1)
    w, ws = weights(96, 100, gen)
    assert ops.int8_mul_mat(w, ws, torch.empty(0, 100, device="cuda", dtype=torch.float16)).shape == (0, 96)
    assert ops.int8_mul_mat(w[:0], ws[:0], torch.empty(5, 100, device="cuda")).shape == (5, 0)
    big = torch.randn(50, 333, device="cuda", generator=gen)
    for x in (big[:, 1:101], big[::7, 5:105], big[:1, :100].expand(4, -1)):
        check_product(ops.int8_mul_mat(w, ws, x), *codes_of(x), w, ws, None, torch.float32)
    # weight rows that are a part of a larger matrix: every third one, and columns from 32 on
    w2, ws2 = weights(96, 256, gen)
    x = big[:, :100]
    check_product(ops.int8_mul_mat(w2[::3, 32:132], ws2[::3].contiguous(), x), *codes_of(x), w2[::3, 32:132], ws2[::3], None, torch.float32)
    # nothing behind the result is written
    out = torch.full((8, 96), 5.0, device="cuda")
    del out
    for bad in (w2[:, 1:101], torch.zeros(96, 100, dtype=torch.int8, device="cuda"), w2.T, w2[:, ::2]):
        with pytest.raises(RuntimeError):
            ops.int8_mul_mat(bad, ws, torch.zeros(3, bad.shape[1], device="cuda"))


@pytest.mark.gpu
@pytest.mark.parametrize("m", [1, 100])
def test_weights_straight_out_of_the_quantizer(ops, m):
    """Weights made by the call ahead in the stream, and overwritten by it: no product reads them too early."""
    gen = torch.Generator(device="cuda").manual_seed(3)
    x = torch.randn(m, 2048, device="cuda", generator=gen, dtype=torch.float32)
    q, qs = ops.int8_quantize(x)
    fs = [torch.randn(2048, 2048, device="cuda", generator=gen) for _ in range(6)]
    got = []
    for f in fs:
        w, ws = ops.int8_quantize(f)
        got.append((ops.int8_mul_mat_prepared(w, ws, q, qs, torch.float32), ops.int8_mul_mat(w, ws, x)))
    for f, (a, b) in zip(fs, got):
        w, ws = codes_of(f)
        check_product(a, *codes_of(x), w, ws, None, torch.float32)
        assert torch.equal(a, b)


@pytest.mark.gpu
def test_streams_graphs_and_threads(ops):
    """Two captured graphs replayed on two streams at once, and eager calls beside them, give what one call alone gives."""
    gen = torch.Generator(device="cuda").manual_seed(9)
    cases = []
    for m, n, k in ((1, 2048, 2048), (40, 1024, 4096), (300, 512, 1024), (3, 2050, 9000), (500, 4096, 8192)):   # (one launch; two; shared; pairs)
        w, ws = weights(n, k, gen)
        x = torch.randn(m, k, device="cuda", generator=gen).to(torch.bfloat16)
        cases.append((w, ws, x, ops.int8_mul_mat(w, ws, x)))
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        side = torch.cuda.Stream()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.stream(side), torch.cuda.graph(g, stream=side):
            outs = [ops.int8_mul_mat(w, ws, x) for w, ws, x, _ in cases]
        graphs.append((g, side, outs))
    for _ in range(5):
        for g, side, outs in graphs:
            for o in outs:
                o.fill_(-1)
        torch.cuda.synchronize()
        for g, side, _ in graphs:
            with torch.cuda.stream(side):
                g.replay()
        eager = [ops.int8_mul_mat(w, ws, x) for w, ws, x, _ in cases]
        torch.cuda.synchronize()
        for got in [outs for _, _, outs in graphs] + [eager]:
            assert all(torch.equal(a, want) for a, (_, _, _, want) in zip(got, cases))


# ---- experts -------------------------------------------------------------------------------------------------


def moe_want(x, w13, s13, w2, s2, weights_, ids, act):
    """(result, tolerance before the last rounding) in float64.  For 16-bit tokens an expert's result is rounded to fp16 once on its way to
    the sum: 2^-11 of itself, or, below fp16's normal numbers, 2^-25 of what it was divided by: powers of two of at most I and at most
    twice the expert's largest scale.  fp32 rounds a hidden value h = act(gate) * up by at most 2^-19 of itself
    (gate and up: 5 * 2^-24 each; the activation's condition number is below 1 + |gate| with |gate| < 100 only where h counts, 2^-19
    covers |gate| < 30): a code within 127 * 2^-18 of a half may go either way, one step of the row's scale times its weight."""
    q, qs = codes_of(x)
    out, room = torch.zeros(x.shape, dtype=torch.float64, device=x.device), torch.zeros(x.shape, dtype=torch.float64, device=x.device)
    half = w13.shape[1] // 2
    for e in range(w13.shape[0]):
        for j in range(ids.shape[1]):
            t = (ids[:, j] == e).nonzero().squeeze(1)
            if t.numel() == 0:
                continue
            both = (q[t] @ w13[e].double().T) * qs[t][:, None] * s13[e].double()
            gate, up = both[:, :half], both[:, half:]
            h = (gate * torch.sigmoid(gate) if act == "silu" else gate * torch.special.ndtr(gate)) * up
            assert float(gate.abs().max()) < 30
            a = h.abs().amax(1, keepdim=True)
            unit = h * 127 / torch.where(a > 0, a, 1.0)
            code = torch.round(unit)
            close = ((unit - torch.floor(unit) - 0.5).abs() < 127 * 2.0 ** -18).double()
            f = (a / 127) * s2[e].double() * weights_[t, j].double()[:, None]
            part = (code @ w2[e].double().T) * f
            out[t] += part
            room[t] += (close @ w2[e].double().abs().T) * f.abs() + 2.0 ** -18 * part.abs()
            if x.dtype != torch.float32:
                room[t] += 2.0 ** -11 * part.abs() + 2.0 ** -25 * half * 2 * float(s2[e].max()) * (a / 127) * weights_[t, j].double().abs()[:, None]
    return out, room


def experts(e, h, i, gen):
    w13, s13 = weights(e * 2 * i, h, gen)
    w2, s2 = weights(e * h, i, gen)
    return w13.unflatten(0, (e, 2 * i)), s13.view(e, 2 * i), w2.unflatten(0, (e, h)), s2.view(e, h)


MOE = [(1, 4, 2, 64, 32), (1, 64, 8, 256, 128), (3, 8, 1, 136, 264), (8, 64, 8, 512, 256), (33, 16, 4, 264, 392), (100, 8, 2, 384, 128), (257, 8, 8, 512, 384),
       (64, 256, 8, 128, 64), (600, 4, 3, 256, 136), (1500, 16, 4, 128, 256),
       (128, 9, 8, 64, 32), (1025, 65, 1, 64, 32), (2049, 64, 4, 64, 32), (1500, 256, 7, 64, 32), (9001, 100, 2, 64, 32), (5, 64, 40, 64, 32), (7, 3, 2, 16408, 40),
       (601, 4, 2, 1160, 40), (600, 3, 1, 2056, 32)]


@pytest.mark.gpu
@pytest.mark.parametrize("t,e,k,h,i", MOE)
@pytest.mark.parametrize("dtype,act", [(torch.bfloat16, "silu"), (torch.float16, "gelu"), (torch.float32, "silu")])
def test_moe(ops, t, e, k, h, i, dtype, act):
    gen = torch.Generator(device="cuda").manual_seed(t + e + h)
    w13, s13, w2, s2 = experts(e, h, i, gen)
    x = torch.randn(t, h, device="cuda", generator=gen).to(dtype)
    weights_, ids = torch.randn(t, e, device="cuda", generator=gen).softmax(-1).topk(k, dim=-1)
    ids = ids.to(torch.int32)
    ids[::5, 0] = -1          # (skipped)
    if t > 4:
        ids[3] = e            # a token without any expert
    y = ops.int8_fused_moe(x, w13, s13, w2, s2, weights_, ids, act)
    want, room = moe_want(x, w13, s13, w2, s2, weights_, ids, act)
    room = room + torch.finfo(dtype).eps / 2 * (want.abs() + room) + TINY[dtype] + 2.0 ** -22 * want.abs()
    assert y.dtype == dtype and bool(((y.double() - want).abs() <= room).all())
    if t > 4:
        assert not bool(y[3].any())
    assert torch.equal(ops.int8_fused_moe(x, w13, s13, w2, s2, weights_, ids, act), y)


@pytest.mark.gpu
def test_moe_all_tokens_to_one_expert_and_the_same_one_twice(ops):
    gen = torch.Generator(device="cuda").manual_seed(2)
    w13, s13, w2, s2 = experts(16, 128, 72, gen)
    x = torch.randn(700, 128, device="cuda", generator=gen)
    weights_ = torch.rand(700, 2, device="cuda", generator=gen)
    ids = torch.full((700, 2), 15, dtype=torch.int32, device="cuda")
    y = ops.int8_fused_moe(x, w13, s13, w2, s2, weights_, ids, "silu")
    want, room = moe_want(x, w13, s13, w2, s2, weights_, ids, "silu")
    assert bool(((y.double() - want).abs() <= room + 2.0 ** -22 * want.abs() + 1e-30).all())
    ids.fill_(-1)
    assert not bool(ops.int8_fused_moe(x, w13, s13, w2, s2, weights_, ids, "silu").any())
    assert ops.int8_fused_moe(x[:0], w13, s13, w2, s2, weights_[:0], ids[:0], "silu").shape == (0, 128)


@pytest.mark.gpu
def test_moe_in_a_graph_with_the_router(ops):
    """Route and experts captured together; replayed on new logits and activations, padded rows among them."""
    gen = torch.Generator(device="cuda").manual_seed(4)
    w13, s13, w2, s2 = experts(32, 256, 128, gen)
    x = torch.randn(48, 256, device="cuda", generator=gen).to(torch.bfloat16)
    logits = torch.randn(48, 32, device="cuda", generator=gen)
    bias = torch.randn(32, device="cuda", generator=gen) * 0.1

    def step():
        weights_, ids = ops.moe_route(logits, 4, scoring="sigmoid", bias=bias, n_group=4, topk_group=2, scale=2.0)
        return ops.int8_fused_moe(x, w13, s13, w2, s2, weights_, ids, "silu"), weights_, ids

    step()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step()
    for i in range(3):
        x.copy_(torch.randn(48, 256, device="cuda", generator=gen))
        logits.copy_(torch.randn(48, 32, device="cuda", generator=gen))
        logits[40 + i:] = float("-inf")
        g.replay()
        torch.cuda.synchronize()
        eager = step()
        assert all(torch.equal(a, b) for a, b in zip(out, eager))
        assert bool((out[2][40 + i:] == -1).all()) and not bool(out[0][40 + i:].any())
        want, room = moe_want(x, w13, s13, w2, s2, out[1], out[2], "silu")
        room = room + 2.0 ** -9 * (want.abs() + room) + 2.0 ** -22 * want.abs() + 1e-30   # (bf16: half of 2^-8)
        assert bool(((out[0].double() - want).abs() <= 2 * room).all())


@pytest.mark.gpu
@pytest.mark.parametrize("t,e,k,h,i", [(1, 8, 4, 256, 128), (40, 8, 2, 264, 136), (600, 4, 3, 128, 64)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_moe_of_16_bit_tokens_sums_in_fp32(ops, t, e, k, h, i, dtype):
    """Nothing between the tokens and the result has fewer than 32 bits: the room of fp32 tokens of the same values, and one rounding to the
    type.  Rows of W2 with scales over eight powers of ten keep their precision too."""
    gen = torch.Generator(device="cuda").manual_seed(t + i)
    w13, s13, w2, _ = experts(e, h, i, gen)
    s2 = 10.0 ** (-8 * torch.rand(e, h, device="cuda", generator=gen))
    s2[:, 0], s2[:, 1] = 1.0, 1e-8
    x = torch.randn(t, h, device="cuda", generator=gen).to(dtype)
    weights_, ids = torch.randn(t, e, device="cuda", generator=gen).softmax(-1).topk(k, dim=-1)
    ids = ids.to(torch.int32)
    y = ops.int8_fused_moe(x, w13, s13, w2, s2, weights_, ids, "silu")
    want, room = moe_want(x.float(), w13, s13, w2, s2, weights_, ids, "silu")
    room = room + torch.finfo(dtype).eps / 2 * (want.abs() + room) + TINY[dtype] + 2.0 ** -22 * want.abs()
    assert y.dtype == dtype and bool(torch.isfinite(want).all())
    assert bool(((y.double() - want).abs() <= room).all())


def rows_of_gates(act, lo, hi, t, i, gen):
    """(x, w13, s13) of two experts whose gates all lie between lo and hi, within 5 %, up halves of both signs."""
    h = 96
    x = 1 + 0.05 * torch.rand(t, h, device="cuda", generator=gen)
    w13, s13 = weights(2 * 2 * i, h, gen)
    w13, s13 = w13.unflatten(0, (2, 2 * i)), s13.view(2, 2 * i)
    w13[:, :i] = -(w13[:, :i].abs().clamp(min=1).clamp(max=127))
    q, qs = codes_of(x)
    mean = (q[0] @ w13[:, :i].double().transpose(1, 2)) * qs[0]
    s13[:, :i] = (torch.linspace(hi, lo, i, device="cuda", dtype=torch.float64) / mean).float()
    return x, w13, s13


@pytest.mark.gpu
@pytest.mark.parametrize("act,lo,hi", [("gelu", -8.0, -3.0), ("gelu", -12.5, -6.0), ("gelu", -2.0, -0.01)])
@pytest.mark.parametrize("t,i", [(3, 64), (70, 136)])
def test_moe_hidden_rows_of_negative_gates(ops, act, lo, hi, t, i):
    """A hidden row goes by its own largest value, so that it needs small activations to be right relative to themselves.

    A gate is D * (q_scale * w_scale) with D below 2^24: the scale, two products, 3 * 2^-24.  What that is in the activation's value is its condition
    number, below 1 + g^2 for g Phi(g) (g phi(g) / Phi(g) is below 1 + g^2 for negative g) and below 1 + |g| for g sigmoid(g).  The activation adds
    2^-20 (of an erfc 2^-21, of an exponential and a reciprocal 2^-23 each, and a few roundings of 2^-24), up and its product 4 * 2^-24."""
    gen = torch.Generator(device="cuda").manual_seed(t + i)
    x, w13, s13 = rows_of_gates(act, lo, hi, t, i, gen)
    w2, s2 = weights(2 * 96, i, gen)
    w2, s2 = w2.unflatten(0, (2, 96)), s2.view(2, 96)
    s2 *= 1e3 / max(1e-30, float(torch.sigmoid(torch.tensor(hi, dtype=torch.float64))))   # (results of ordinary size)
    ids = (torch.arange(t, device="cuda") % 2).to(torch.int32)[:, None].contiguous()
    y = ops.int8_fused_moe(x, w13, s13, w2, s2, torch.ones(t, 1, device="cuda"), ids, act)
    q, qs = codes_of(x)
    for e in range(2):
        s = ids[:, 0] == e
        both = (q[s] @ w13[e].double().T) * qs[s][:, None] * s13[e].double()
        g, up = both[:, :i], both[:, i:]
        assert bool((g < 0.9 * hi).all()) and bool((g > 1.1 * lo).all())
        h = (g * torch.sigmoid(g) if act == "silu" else g * torch.special.ndtr(g)) * up
        rel = (1 + (g * g if act == "gelu" else g.abs())) * 3 * 2.0 ** -24 + 2.0 ** -20 + 2.0 ** -22
        a, top = h.abs().max(1, keepdim=True)
        unit = h * 127 / a
        close = ((unit - torch.floor(unit) - 0.5).abs() < unit.abs() * (rel + rel.gather(1, top)) + 2.0 ** -30).double()
        f = (a / 127) * s2[e].double()
        want = (torch.round(unit) @ w2[e].double().T) * f
        room = (close @ w2[e].double().abs().T) * f + want.abs() * (rel.gather(1, top) + 8 * 2.0 ** -24)
        off = (y[s].double() - want).abs()
        assert bool((off <= room).all()), (float((off / want.abs().amax()).max()), float((room / want.abs().amax()).max()))


@pytest.mark.gpu
@pytest.mark.parametrize("act,sign,size", [("silu", -1, 2.0 ** -13), ("silu", -1, 2.0 ** -16), ("silu", 1, 2.0 ** -14), ("gelu", -1, 2.0 ** -16), ("gelu", 1, 2.0 ** -16)])
def test_moe_activation_of_exact_gates(ops, act, sign, size):
    """Scales that are powers of two and sums below 2^24: gates (of a size up to 75, 10 or 38) and up halves reach the activation without a rounding.
    What is left is the activation's 2^-21 (silu: an exponential and a reciprocal to 2^-23 each, three roundings of 2^-24) or 2^-20 (gelu), up's product, the
    row's scale a / 127, and four roundings of the down product, 2^-24 each."""
    gen = torch.Generator(device="cuda").manual_seed(int(1 / size) + sign)
    t, h, i = 40, 96, 72
    x = torch.randint(60, 128, (t, h), device="cuda", generator=gen).float()
    x[:, 5] = 127                                              # (codes are the values, the scale is 1)
    buf = torch.randint(-127, 128, (1, 2 * i, h), device="cuda", generator=gen)
    big = 30 + torch.arange(i, device="cuda")[:, None] // 2    # (gate rows of different sizes)
    buf[0, :i] = sign * (big - torch.randint(0, 10, (i, h), device="cuda", generator=gen))
    w13, s13 = buf.to(torch.int8), torch.full((1, 2 * i), size, device="cuda")
    w2 = torch.randint(-127, 128, (1, 64 + 32, 80), device="cuda", generator=gen).to(torch.int8)[:, :, :i]
    s2 = torch.full((1, h), 2.0 ** 20, device="cuda")
    y = ops.int8_fused_moe(x, w13, s13, w2, s2, torch.ones(t, 1, device="cuda"), torch.zeros(t, 1, dtype=torch.int32, device="cuda"), act)
    both = (x.double() @ w13[0].double().T) * size
    g, up = both[:, :i], both[:, i:]
    assert float(g.abs().max()) < 76 and bool((g.abs() > 0.1).all())
    hidden = (g * torch.sigmoid(g) if act == "silu" else g * torch.special.ndtr(g)) * up
    rel = 2.0 ** (-21 if act == "silu" else -20) + 2.0 ** -24
    a = hidden.abs().amax(1, keepdim=True)
    unit = hidden * 127 / a
    close = ((unit - torch.floor(unit) - 0.5).abs() < 127 * 2 * rel).double()
    f = a / 127 * 2.0 ** 20
    want = (torch.round(unit) @ w2[0].double().T) * f
    room = (close @ w2[0].double().abs().T) * f + want.abs() * (rel + 5 * 2.0 ** -24)
    off = (y.double() - want).abs()
    assert bool((off <= room).all()), (float((off / want.abs().amax()).max()), float((room / want.abs().amax()).max()))


class Guarded:
    """A buffer between two stretches of a pattern that have to be found again; `skew` elements behind a multiple of 256 bytes."""

    def __init__(self, n, dtype, skew=0):
        size = torch.empty(0, dtype=dtype).element_size()
        self.front, self.bytes = 1024 + skew * size, n * size
        self.all = torch.full((self.front + self.bytes + 8192,), 0xA5, dtype=torch.uint8, device="cuda")
        self.p = ctypes.c_void_p(self.all.data_ptr() + self.front)
        self.view = self.all[self.front:self.front + self.bytes].view(dtype)

    def check(self, what):
        clean = bool((self.all[:self.front] == 0xA5).all()) and bool((self.all[self.front + self.bytes:] == 0xA5).all())
        assert clean, f"{what}: written beside"


@pytest.mark.gpu
@pytest.mark.parametrize("m,n,k", [(1, 131, 96), (1, 4096, 2048), (5, 2050, 1000), (8, 1, 40), (3, 2050, 9000), (20, 2100, 14000), (33, 127, 300), (257, 130, 640),
                                   (520, 4225, 1030), (450, 9000, 528), (1000, 333, 144)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_nothing_is_written_beside_results(native_libs, m, n, k, dtype):
    from gguf_b200 import capi

    lib, code, stream = capi.lib(), DTYPES.index(dtype), ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
    gen = torch.Generator(device="cuda").manual_seed(m + n)
    w, ws = weights(n, k, gen)
    x = torch.randn(m, k, device="cuda", generator=gen).to(dtype)
    qwant, swant = codes_of(x)
    pitch = (k + 15) // 16 * 16
    q, qs = Guarded(m * pitch, torch.int8), Guarded(m, torch.float32, 1)
    assert lib.gguf_b200_int8_quantize(x.data_ptr(), code, k, q.p, pitch, qs.p, m, k, stream) == 0
    q.check("codes")
    qs.check("scales")
    assert torch.equal(q.view.view(m, pitch)[:, :k].double(), qwant)
    assert bool((q.view.view(m, pitch)[:, k:] == torch.tensor(0xA5, dtype=torch.uint8).view(torch.int8)).all())   # (nor behind the values of a row)
    room = lib.gguf_b200_int8_scratch_bytes(m, k)
    for skew in (0, 1):       # (rows that 16-byte stores can be made to, and others)
        y, scratch = Guarded(m * n, dtype, skew), Guarded(room, torch.uint8)
        assert lib.gguf_b200_int8_mul_mat(w.data_ptr(), w.stride(0), ws.data_ptr(), x.data_ptr(), k, None, y.p, scratch.p, room, 0, code, m, n, k, stream) == 0
        y.check("product")
        scratch.check("workspace")
        check_product(y.view.view(m, n), qwant, swant, w, ws, None, dtype)
        z = Guarded(m * n, dtype, skew)
        assert lib.gguf_b200_int8_mul_mat_prepared(w.data_ptr(), w.stride(0), ws.data_ptr(), q.p, pitch, qs.p, None, z.p, 0, code, m, n, k, stream) == 0
        z.check("prepared")
        assert torch.equal(z.view, y.view)
    assert capi.last_status() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("t,e,k,h,i", [(1, 5, 3, 72, 40), (33, 16, 4, 264, 392), (1025, 65, 1, 64, 32), (2049, 64, 4, 64, 32), (300, 8, 2, 1160, 136)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_nothing_is_written_beside_the_results_of_experts(native_libs, t, e, k, h, i, dtype):
    from gguf_b200 import capi

    lib, code, stream = capi.lib(), DTYPES.index(dtype), ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
    gen = torch.Generator(device="cuda").manual_seed(t + h)
    w13, s13, w2, s2 = experts(e, h, i, gen)
    x = torch.randn(t, h, device="cuda", generator=gen).to(dtype)
    logits = torch.randn(t, e, device="cuda", generator=gen)
    rw, ids = Guarded(t * k, torch.float32, 1), Guarded(t * k, torch.int32, 3)
    assert lib.gguf_b200_moe_route(logits.data_ptr(), 0, e, None, rw.p, ids.p, t, e, k, 1, 1, 1, 1, 1.0, stream) == 0
    rw.check("weights")
    ids.check("ids")
    ids.view[::7] = -1
    room = lib.gguf_b200_int8_moe_workspace_bytes(t, k, e, h, i)
    y, scratch = Guarded(t * h, dtype), Guarded(room, torch.uint8)
    assert lib.gguf_b200_int8_fused_moe(x.data_ptr(), h, w13.data_ptr(), w13.stride(1), s13.data_ptr(), w2.data_ptr(), w2.stride(1), s2.data_ptr(), y.p, ids.p, rw.p,
                                        scratch.p, room, code, 1, t, k, e, h, i, stream) == 0
    y.check("result")
    scratch.check("workspace")
    assert torch.equal(y.view.view(t, h), capi.int8_fused_moe(x, w13, s13, w2, s2, rw.view.clone().view(t, k), ids.view.clone().view(t, k)))
    assert capi.last_status() == 0


# ---- refusals ------------------------------------------------------------------------------------------------


def test_c_abi_refuses_before_any_launch(native_libs):
    from gguf_b200 import capi

    lib = capi.lib()
    p, odd, null = ctypes.c_void_p(4096), ctypes.c_void_p(4104), None
    q = lib.gguf_b200_int8_quantize
    assert q(p, 7, 64, p, 64, p, 1, 64, null) == -2
    assert q(p, 1, 64, p, 64, p, -1, 64, null) == -3 and q(p, 1, 64, p, 64, p, 1, 0, null) == -3
    assert q(null, 1, 64, p, 64, p, 1, 64, null) == -4 and q(p, 1, 64, odd, 64, p, 1, 64, null) == -4
    assert q(p, 1, 64, p, 48, p, 1, 64, null) == -4 and q(p, 1, 64, p, 72, p, 1, 64, null) == -4 and q(p, 1, 64, p, 64, null, 1, 64, null) == -4
    assert q(ctypes.c_void_p(4097), 1, 64, p, 64, p, 1, 64, null) == -4 and q(ctypes.c_void_p(4098), 0, 64, p, 64, p, 1, 64, null) == -4
    assert q(null, 1, 64, null, 64, null, 0, 64, null) == 0
    m = lib.gguf_b200_int8_mul_mat
    assert lib.gguf_b200_int8_scratch_bytes(3, 100) == 512 + 256 and lib.gguf_b200_int8_scratch_bytes(0, 100) == 0
    assert m(p, 64, p, p, 64, null, p, p, 1 << 20, 0, 9, 1, 8, 64, null) == -2
    assert m(p, 64, p, p, 64, null, p, p, 1 << 20, 0, 1, 1, 8, 0, null) == -3
    assert m(p, 131072, p, p, 131072, null, p, p, 1 << 20, 0, 1, 1, 8, 131072, null) == -7
    assert m(odd, 64, p, p, 64, null, p, p, 1 << 20, 0, 1, 1, 8, 64, null) == -4 and m(p, 72, p, p, 64, null, p, p, 1 << 20, 0, 1, 1, 8, 64, null) == -4
    assert m(p, 64, null, p, 64, null, p, p, 1 << 20, 0, 1, 1, 8, 64, null) == -4 and m(p, 64, p, p, 64, null, p, null, 0, 0, 1, 1, 8, 64, null) == -4
    assert m(p, 64, p, p, 64, null, p, p, 16, 0, 1, 1, 8, 64, null) == -5
    assert m(p, 64, p, p, 64, null, p, p, 0, 0, 1, 0, 8, 64, null) == 0
    pr = lib.gguf_b200_int8_mul_mat_prepared
    assert pr(p, 64, p, odd, 64, p, null, p, 0, 1, 1, 8, 64, null) == -4 and pr(p, 64, p, p, 64, null, null, p, 0, 1, 1, 8, 64, null) == -4
    moe = lib.gguf_b200_int8_fused_moe
    room = lib.gguf_b200_int8_moe_workspace_bytes(4, 2, 8, 64, 64)
    assert room > 0 and lib.gguf_b200_int8_moe_workspace_bytes(4, 2, 257, 64, 64) == 0

    def call(w13=p, ld13=64, act=1, dtype=1, top_k=2, e=8, h=64, i=64, ws=room, ids=p, y=p):
        return moe(p, 64, w13, ld13, p, p, 64, p, y, ids, p, p, ws, dtype, act, 4, top_k, e, h, i, null)

    assert call(act=3) == -3 and call(h=60) == -3 and call(i=36) == -3 and call(top_k=0) == -3 and call(e=0) == -3
    assert call(dtype=5) == -2 and call(e=257) == -7 and call(w13=odd) == -4 and call(ld13=72) == -4 and call(ids=null) == -4 and call(y=odd) == -4
    assert call(ws=room - 1) == -5 and call(top_k=257) == -7


def test_c_abi_refuses_pointers_off_their_elements(native_libs):
    """Every argument that a kernel reads or writes by its elements, one at a time, and a negative distance between rows."""
    from gguf_b200 import capi

    lib = capi.lib()
    p, off1, off2 = ctypes.c_void_p(4096), ctypes.c_void_p(4097), ctypes.c_void_p(4098)
    q = lib.gguf_b200_int8_quantize
    assert q(p, 1, 64, p, 64, off2, 1, 64, None) == -4

    def mul_mat(w_scales=p, bias=p, dtype=1, m=1, ldx=64):
        return lib.gguf_b200_int8_mul_mat(p, 64, w_scales, p, ldx, bias, p, p, 1 << 20, 0, dtype, m, 8, 64, None)

    def prepared(w_scales=p, q_scales=p, bias=p, dtype=1):
        return lib.gguf_b200_int8_mul_mat_prepared(p, 64, w_scales, p, 64, q_scales, bias, p, 0, dtype, 1, 8, 64, None)

    for m in (1, 40):
        assert mul_mat(w_scales=off2, m=m) == -4 and mul_mat(bias=off1, m=m) == -4 and mul_mat(bias=off1, dtype=2, m=m) == -4 and mul_mat(bias=off2, dtype=0, m=m) == -4
        assert mul_mat(ldx=-64, m=m) == -3
    assert prepared(w_scales=off2) == -4 and prepared(q_scales=off2) == -4 and prepared(bias=off1) == -4 and prepared(bias=off2, dtype=0) == -4
    room = lib.gguf_b200_int8_moe_workspace_bytes(4, 2, 8, 64, 64)

    def moe(ldx=64, s13=p, s2=p, ids=p, weights=p):
        return lib.gguf_b200_int8_fused_moe(p, ldx, p, 64, s13, p, 64, s2, p, ids, weights, p, room, 1, 1, 4, 2, 8, 64, 64, None)

    assert moe(ldx=-1) == -3 and moe(s13=off2) == -4 and moe(s2=off2) == -4 and moe(ids=off2) == -4 and moe(weights=off2) == -4

    def route(bias=None, weights=p, ids=p):
        return lib.gguf_b200_moe_route(p, 1, 64, bias, weights, ids, 4, 64, 8, 1, 1, 1, 1, 1.0, None)

    assert route(bias=off2) == -4 and route(weights=off2) == -4 and route(ids=off2) == -4


def test_shapes_under_tracing(ops):
    from torch._subclasses.fake_tensor import FakeTensorMode

    with FakeTensorMode():
        dev = "cuda" if torch.cuda.is_available() else "meta"
        x = torch.empty(5, 100, device=dev, dtype=torch.bfloat16)
        q, s = torch.ops._C_gguf.int8_quantize(x)
        assert q.shape == (5, 100) and q.stride() == (112, 1) and q.dtype == torch.int8 and s.shape == (5,) and s.dtype == torch.float32
        w = torch.empty(7, 100, device=dev, dtype=torch.int8)
        assert torch.ops._C_gguf.int8_mul_mat(w, s, x, None).shape == (5, 7)
        y = torch.ops._C_gguf.int8_mul_mat_prepared(w, s, q, s, None, torch.float16)
        assert y.shape == (5, 7) and y.dtype == torch.float16
        assert torch.ops._C_gguf.int8_fused_moe(x, w, s, w, s, s, s, 1).shape == x.shape
        a, b = torch.ops._C_gguf.moe_route(x, None, 4, 1, 1, 1, True, 1.0)
        assert a.shape == b.shape == (5, 4) and a.dtype == torch.float32 and b.dtype == torch.int32


@pytest.mark.gpu
def test_refuses_what_it_cannot_take(ops):
    w, ws = torch.zeros(32, 64, dtype=torch.int8, device="cuda"), torch.ones(32, device="cuda")
    x = torch.zeros(3, 64, device="cuda")
    for args in ((w.to(torch.uint8), ws, x), (w, ws[:-1], x), (w, ws.double(), x), (w, ws, x[:, :48]), (w, ws, x.double()), (w, ws, x[0]), (w[0], ws, x),
                 (w, ws.cpu(), x), (w.cpu(), ws, x), (w, ws, x, torch.ones(31, device="cuda")), (w, ws, x, torch.ones(32, device="cuda", dtype=torch.float16)),
                 (w, ws, x.T.contiguous().T)):
        with pytest.raises((RuntimeError, NotImplementedError)):
            ops.int8_mul_mat(*args)
    with pytest.raises(RuntimeError):
        ops.int8_quantize(torch.zeros(3, 4, 5, device="cuda"))
    with pytest.raises(RuntimeError):
        ops.int8_quantize(torch.zeros(3, 4, device="cuda", dtype=torch.int32))
    with pytest.raises(KeyError):
        ops.int8_fused_moe(x, w[None], ws[None], w[None], ws[None], ws, ws, "relu")
