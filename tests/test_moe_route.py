"""The expert router against its definition in 64 bits.  Ids are compared for equality.  A weight is computed in fp32: an exponential (2 units in the last
place, 2^-22; the rounding error of x - max is carried along), a sum and a quotient or two (2^-24 each), the sum of the row's weights
(their errors, and five roundings of 2^-24), a product with the scale: below 2^-20 in all.  The sum of a softmax over up to 512 experts adds up to 21 roundings of 2^-24 where it is needed: 2^-19."""
import ctypes

import pytest
import torch

INF, NAN = float("inf"), float("nan")
DTYPES = [torch.float32, torch.float16, torch.bfloat16]


@pytest.fixture(scope="module")
def ops(native_libs):
    from vllm_gguf_plugin import ops

    return ops


def route(logits, top_k, scoring="softmax", bias=None, n_group=1, topk_group=1, renormalize=True, scale=1.0):
    """A row at a time, from the definition."""
    ids, weights = [], []
    bias = [0.0] * logits.shape[1] if bias is None else (None, bias.double().tolist())[1]
    given = any(b != 0 for b in bias)
    for row in logits.double().cpu():
        x = [min(v, 3.4028234663852886e38) if v == v else -INF for v in row.tolist()]
        live = [v > -INF for v in x]
        t = torch.tensor(x, dtype=torch.float64)
        s = (torch.softmax(t, 0) if any(live) else torch.zeros_like(t)) if scoring == "softmax" else torch.sigmoid(t)
        s = s.tolist()
        choice = [(s[e] + bias[e] if given else x[e]) if live[e] else -INF for e in range(len(x))]
        choice = [c if c == c else -INF for c in choice]
        per = len(x) // n_group
        if n_group > 1:
            score = []
            for g in range(n_group):
                best = sorted((c for c in choice[g * per:(g + 1) * per] if c > -INF), reverse=True)
                score.append(-INF if not best else sum(best[:2]) if given else best[0])
            keep = sorted(range(n_group), key=lambda g: (-score[g], g))[:topk_group]
            choice = [c if e // per in keep else -INF for e, c in enumerate(choice)]
        order = [e for e in sorted(range(len(x)), key=lambda e: (-choice[e], e)) if choice[e] > -INF][:top_k]
        w = [s[e] for e in order]
        total = sum(w)
        if renormalize and total > 0:
            w = [v / total for v in w]
        ids.append(order + [-1] * (top_k - len(order)))
        weights.append([v * scale for v in w] + [0.0] * (top_k - len(order)))
    return torch.tensor(weights, dtype=torch.float64), torch.tensor(ids, dtype=torch.int32)


def check(got, want, summed=False):
    w, ids = got
    assert w.dtype == torch.float32 and ids.dtype == torch.int32 and w.is_contiguous() and ids.is_contiguous()
    assert torch.equal(ids.cpu(), want[1])
    assert bool(((w.cpu().double() - want[0]).abs() <= 2.0 ** (-19 if summed else -20) * want[0].abs() + 2.0 ** -149).all())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("t,e,k,groups,topk_group", [(1, 1, 1, 1, 1), (1, 64, 8, 1, 1), (5, 7, 7, 1, 1), (33, 60, 4, 4, 2), (50, 64, 6, 8, 3), (9, 128, 16, 4, 4),
                                                     (21, 160, 6, 8, 3), (40, 256, 8, 8, 4), (3, 512, 32, 32, 8), (2, 300, 10, 3, 2), (300, 32, 2, 16, 1)])
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("with_bias", [False, True])
def test_route(ops, dtype, t, e, k, groups, topk_group, scoring, with_bias):
    gen = torch.Generator(device="cuda").manual_seed(t + e)
    logits = (torch.randn(t, e, device="cuda", generator=gen) * 2).to(dtype)
    bias = torch.randn(e, device="cuda", generator=gen) * 0.2 if with_bias else None
    for renormalize, scale in ((True, 1.0), (False, 2.5)):
        kw = dict(scoring=scoring, bias=bias, n_group=groups, topk_group=topk_group, renormalize=renormalize, scale=scale)
        check(ops.moe_route(logits, k, **kw), route(logits, k, **kw), scoring == "softmax" and not renormalize)


@pytest.mark.gpu
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("with_bias", [False, True])
@pytest.mark.parametrize("groups", [1, 4])
def test_route_ties_masks_and_extremes(ops, scoring, with_bias, groups):
    e, k = 32, 12
    low = torch.finfo(torch.float32).min
    rows = [torch.zeros(e), torch.full((e,), -INF), torch.full((e,), NAN), torch.full((e,), INF), torch.full((e,), low), torch.full((e,), 3e38)]
    r = torch.arange(e, dtype=torch.float32) % 3
    rows.append(r)                                            # many equals
    rows += [torch.where(r > 0, -INF, 1.0), torch.where(r > 0, NAN, 1.0), torch.where(r > 1, INF, 0.5), torch.where(r > 1, low, -1.0)]
    one = torch.full((e,), -INF)
    one[17] = -3.0
    rows.append(one)                                          # one expert left
    two = torch.full((e,), -INF)
    two[30], two[2] = 1.0, -1000.0
    rows.append(two)
    rows.append(torch.linspace(-1, 1, e) * 80)
    rows.append(torch.where(r > 0, 0.0, -0.0))                # zeros of both signs are equal
    logits = torch.stack(rows).cuda()
    bias = None
    if with_bias:
        bias = torch.zeros(e, device="cuda")
        bias[::5], bias[3], bias[9], bias[20], bias[21] = -0.5, INF, -INF, NAN, 0.25
    for topk_group in range(max(1, -(-k * groups // e)), groups + 1):
        for renormalize in (True, False):
            kw = dict(scoring=scoring, bias=bias, n_group=groups, topk_group=topk_group, renormalize=renormalize)
            check(ops.moe_route(logits, k, **kw), route(logits, k, **kw), scoring == "softmax" and not renormalize)


@pytest.mark.gpu
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
def test_route_choices_next_to_one_another(ops, scoring):
    """Choices that fp32 cannot tell apart: the order is that of fp64."""
    gen = torch.Generator().manual_seed(0)
    e = 64
    logits = torch.randn(200, e, generator=gen)
    s = torch.softmax(logits.double(), -1) if scoring == "softmax" else torch.sigmoid(logits.double())
    bias = (0.75 - s[0]).float()                              # in row 0 every choice is 0.75 up to the rounding of the bias
    logits[1::2] = logits[0] + torch.randn(100, e, generator=gen) * 1e-7
    kw = dict(scoring=scoring, bias=bias.cuda(), n_group=8, topk_group=4)
    check(ops.moe_route(logits.cuda(), 8, **kw), route(logits, 8, **{**kw, "bias": bias}))


@pytest.mark.gpu
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("with_bias", [False, True])
@pytest.mark.parametrize("e,k", [(60, 8), (300, 32), (512, 5), (33, 32)])
def test_route_runs_of_equals(ops, scoring, with_bias, e, k):
    """Runs of equal, or nearly equal, choices that begin before the last place and end behind it, of a few experts and of more than a warp has lanes."""
    gen = torch.Generator().manual_seed(e + k)
    rows = []
    for run in (2, 3, 9, 31, 32, 33, 34, 40, e):
        for start in (0, 1, k - 1, k, max(0, k - run), max(0, k + 1 - run)):
            row = torch.linspace(3, -3, e) + 1e-3 * torch.rand(e, generator=gen)
            row[start:start + run] = row[min(start, e - 1)]
            row[e - 3:] = torch.where(torch.rand(3, generator=gen) > 0.5, -INF, row[e - 3:])
            rows.append(row[torch.randperm(e, generator=gen)])
            rows.append(torch.nextafter(rows[-1], torch.tensor(9.0)).where(torch.rand(e, generator=gen) > 0.5, rows[-1]))
    logits = torch.stack(rows)
    logits[3, ::2] = INF
    logits[5, ::3], logits[5, 1::3] = INF, torch.finfo(torch.float32).max
    bias = torch.full((e,), 0.125) if with_bias else None
    for renormalize in (True, False):
        kw = dict(scoring=scoring, n_group=1, topk_group=1, renormalize=renormalize)
        check(ops.moe_route(logits.cuda(), k, bias=None if bias is None else bias.cuda(), **kw), route(logits, k, bias=bias, **kw),
              scoring == "softmax" and not renormalize)


@pytest.mark.gpu
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("k", [1, 4, 7])
def test_route_experts_far_below_the_best(ops, scoring, k):
    """A bias that keeps the row's best experts out: what is chosen lies 20 to 200 below them, and its weights still add up to one."""
    e = 32
    rows = []
    for top, drop, step in ((0.0, 20.0, 1.0), (0.0, 69.0, 1.0), (0.0, 80.0, 1.0), (5.0, 95.0, 0.5), (0.0, 110.0, 3.0), (-70.0, 20.0, 0.25), (-100.0, 90.0, 1.0), (0.0, 200.0, 10.0)):
        row = top - drop - step * torch.arange(e, dtype=torch.float32)
        row[0] = top
        rows += [row, row.flip(0), torch.where(torch.arange(e) % 5 == 4, -INF, row)]
    logits = torch.stack(rows)
    for value in (-INF, -2.0):
        bias = torch.zeros(e)
        bias[0] = bias[e - 1] = value
        for groups, topk_group in ((1, 1), (4, 2)):
            if groups > 1:
                bias[:8] -= 3.0                               # (the best expert's group is out)
            kw = dict(scoring=scoring, n_group=groups, topk_group=topk_group)
            got = ops.moe_route(logits.cuda(), k, bias=bias.cuda(), **kw)
            check(got, route(logits, k, bias=bias, **kw))
            assert bool(((got[0].double().sum(1) - 1).abs() < 2.0 ** -20).all())
            check(ops.moe_route(logits.cuda(), k, bias=bias.cuda(), renormalize=False, **kw), route(logits, k, bias=bias, renormalize=False, **kw), scoring == "softmax")


@pytest.mark.gpu
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("e,groups,topk_group", [(64, 8, 4), (256, 8, 3), (60, 4, 1), (512, 32, 7)])
@pytest.mark.parametrize("size", [1.0, 100.0, 1e5])
def test_route_groups_of_choices_that_cancel(ops, scoring, e, groups, topk_group, size):
    """A bias of both signs: a group's two best choices are large and their sum is small, so that what they were rounded by is more than what is between groups."""
    gen = torch.Generator().manual_seed(e + groups)
    logits = torch.randn(200, e, generator=gen) * torch.tensor([1.0, 0.1, 0.01, 0.001]).repeat(50)[:, None]
    per = e // groups
    bias = torch.full((e,), -size)
    bias[1::per] = size
    bias[per // 2:2 * per:per] -= size / 2                    # (groups that are plainly out, or in)
    bias[3 * per:4 * per] -= 1e9 if size == 1.0 else 0.0
    kw = dict(scoring=scoring, n_group=groups, topk_group=topk_group)
    check(ops.moe_route(logits.cuda(), 4, bias=bias.cuda(), **kw), route(logits, 4, bias=bias, **kw))


@pytest.mark.gpu
def test_route_strides_streams_and_empty(ops):
    gen = torch.Generator(device="cuda").manual_seed(8)
    big = torch.randn(30, 201, device="cuda", generator=gen)
    for logits in (big[:, 1:65], big[::4, 7:71], big[:1, :64].expand(5, -1), big[2:3, 3:67]):
        check(ops.moe_route(logits, 6), route(logits, 6))
    w, ids = ops.moe_route(big[:0], 4)
    assert w.shape == ids.shape == (0, 4)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = ops.moe_route(big, 5, scoring="sigmoid")
    side.synchronize()
    check(got, route(big, 5, scoring="sigmoid"))


@pytest.mark.gpu
def test_route_large(ops):
    gen = torch.Generator(device="cuda").manual_seed(1)
    logits, bias = torch.randn(9001, 256, device="cuda", generator=gen), torch.randn(256, device="cuda", generator=gen) * 0.1
    kw = dict(scoring="sigmoid", n_group=8, topk_group=4, scale=2.5)
    w, ids = ops.moe_route(logits, 8, bias=bias, **kw)
    pick = torch.arange(0, 9001, 61)
    check((w[pick], ids[pick]), route(logits[pick], 8, bias=bias, **kw))
    assert bool((ids >= 0).all()) and bool((ids < 256).all()) and bool(((w.double().sum(1) - 2.5).abs() < 1e-5).all())


def test_c_abi_refuses_before_any_launch(native_libs):
    from gguf_b200 import capi

    lib = capi.lib()
    p = ctypes.c_void_p(4096)

    def call(dtype=0, logits=p, weights=p, ids=p, tokens=4, e=64, k=8, groups=8, topk_group=2, scoring=1):
        return lib.gguf_b200_moe_route(logits, dtype, 64, None, weights, ids, tokens, e, k, groups, topk_group, scoring, 1, 1.0, None)

    assert call(dtype=3) == -2
    for bad in (dict(tokens=-1), dict(e=0), dict(k=0), dict(groups=0), dict(topk_group=0), dict(scoring=0), dict(scoring=3), dict(groups=7), dict(topk_group=9),
                dict(k=17)):
        assert call(**bad) == -3, bad
    assert call(e=520, groups=1, topk_group=1) == -7 and call(k=33, topk_group=8) == -7 and call(groups=64, topk_group=64) == -7
    assert call(logits=ctypes.c_void_p(4098)) == -4 and call(logits=None) == -4 and call(weights=None) == -4 and call(ids=None) == -4
    assert call(tokens=0, logits=None) == 0


def test_refusals_of_the_operator(ops):
    x = torch.zeros(2, 8)
    with pytest.raises(NotImplementedError, match="scoring"):
        ops.moe_route(x, 2, scoring="relu")
    with pytest.raises(NotImplementedError):
        ops.moe_route(x, 2)      # no CPU kernel, and no fallback


@pytest.mark.gpu
def test_refusals_on_the_device(ops):
    x = torch.zeros(2, 8, device="cuda")
    for kw in (dict(top_k=9), dict(top_k=0), dict(top_k=2, n_group=3), dict(top_k=5, n_group=2, topk_group=1), dict(top_k=2, n_group=2, topk_group=3),
               dict(top_k=2, bias=torch.zeros(7, device="cuda")), dict(top_k=2, bias=torch.zeros(8))):
        with pytest.raises(RuntimeError):
            ops.moe_route(x, kw.pop("top_k"), **kw)
    for bad in (x[0], x.long(), x.T.contiguous().T):
        with pytest.raises((RuntimeError, NotImplementedError)):
            ops.moe_route(bad, 1)
