"""k3x_hip_route against a plain implementation in 64 bits, at the sizes and
masks where it can go wrong.

Scores are rounded where the operator documents it (the layer router's steps
for sigmoid, one rounding of the double quotient for softmax), so ids are
compared exactly.  A weight is a score of one rounding over a sum of up to 64
terms of one rounding each and times the scale: at most (2 + 64 + 2) * 2^-24 of
its value with the fp32 sum, (1 + 3) * 2^-24 with the double one; a sigmoid
score itself is within 4 * 2^-24 of the 64-bit one (exp, sum and quotient
rounded once each; the sum's is at most doubled by 1 / (1 + t))."""
from __future__ import annotations

import math

import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")
DEV = "cuda:0"


@pytest.fixture(scope="module")
def hip():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    import k3x_amd
    ctx = k3x_amd.Context(0)
    yield k3x_amd, ctx
    ctx.close()


def gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def scores_of(logits, softmax):
    l = logits.double().cpu()
    if softmax:
        e = torch.exp(l - l.amax(1, keepdim=True))
        return (e / e.sum(1, keepdim=True)).float()
    return 1.0 / (1.0 + torch.exp(-l).float())


def plain(logits, bias, K, softmax=False, groups=1, top_groups=1, top2=True, renorm=True,
          scale=1.0):
    """ids and 64-bit weights of the rounded scores, row by row in Python."""
    s = scores_of(logits, softmax)
    a = s if bias is None else s + bias.cpu()
    ids = torch.empty((len(s), K), dtype=torch.int64)
    n = s.shape[1] // groups
    for t, row in enumerate(a.tolist()):
        kept = range(groups)
        if top_groups < groups:
            rank = []
            for g in kept:
                part = sorted(row[g * n:(g + 1) * n], reverse=True)
                v = part[0]
                if top2 and n > 1:
                    v = float(torch.tensor(part[0]) + torch.tensor(part[1]))
                rank.append((-v, g))
            kept = sorted(g for _, g in sorted(rank)[:top_groups])
        among = [(-row[e], e) for g in kept for e in range(g * n, (g + 1) * n)]
        ids[t] = torch.tensor([e for _, e in sorted(among)[:K]])
    w = s.double().gather(1, ids)
    if renorm:
        w = w / w.sum(1, keepdim=True)
    return ids, w * scale


def call(hip, logits, bias, K, softmax=False, groups=1, top_groups=1, top2=True,
         renorm="float", scale=1.0):
    k3x, ctx = hip
    T, E = logits.shape
    p = k3x.make_route_params(
        T, E, K, scoring=k3x.SCORE_SOFTMAX if softmax else k3x.SCORE_SIGMOID,
        renorm=dict(float=k3x.RENORM_FLOAT, double=k3x.RENORM_DOUBLE, none=k3x.RENORM_NONE)[renorm],
        routed_scale=scale, groups=groups, top_groups=top_groups,
        group_score=k3x.GROUP_TOP2 if top2 else k3x.GROUP_MAX)
    ids = torch.full((T, K), -7, dtype=torch.int32, device=DEV)
    w = torch.full((T, K), -7.0, device=DEV)
    st = k3x.route(ctx, p, logits, ids, w, bias=bias)
    return st, ids, w


def check(hip, logits, bias, K, **kw):
    k3x, ctx = hip
    print(f"[gpu-test] route {tuple(logits.shape)} {logits.dtype} K={K} {kw}", flush=True)
    st, ids, w = call(hip, logits, bias, K, **kw)
    assert st == 0
    assert ctx.synchronize() == 0
    renorm = kw.pop("renorm", "float")
    want_ids, want = plain(logits, bias, K, renorm=renorm != "none", **kw)
    assert torch.equal(ids.cpu().long(), want_ids)
    n = {"float": 4 + K, "double": 4, "none": 2}[renorm]
    err = (w.cpu().double() - want).abs()
    assert (err <= n * 2.0 ** -24 * want.abs() + 2.0 ** -149).all(), float((err / want).max())


@pytest.mark.parametrize("T,E,K", [(1, 1, 1), (1, 16, 4), (2, 384, 16), (3, 63, 5), (5, 64, 64),
                                   (4, 65, 1), (7, 200, 8), (2, 896, 16), (3, 1024, 64),
                                   (2, 1025, 9), (2, 4096, 33), (131, 256, 8), (300, 512, 16)])
@pytest.mark.parametrize("softmax", [False, True], ids=["sigmoid", "softmax"])
@pytest.mark.parametrize("renorm", ["float", "double", "none"])
def test_sizes(hip, T, E, K, softmax, renorm):
    g = gen(T * E + K)
    logits = torch.randn((T, E), device=DEV, generator=g) * 2
    bias = torch.randn((E,), device=DEV, generator=g) * (0.01 if softmax else 0.1)
    check(hip, logits, bias, K, softmax=softmax, renorm=renorm, scale=2.5)
    check(hip, logits.bfloat16(), None, K, softmax=softmax, renorm=renorm)


@pytest.mark.parametrize("E,groups,top_groups,K", [(256, 8, 4, 8), (384, 4, 1, 16), (64, 64, 9, 9),
                                                   (60, 4, 3, 13), (896, 7, 2, 16), (33, 3, 2, 5),
                                                   (4096, 2, 1, 64), (128, 64, 2, 4)])
@pytest.mark.parametrize("top2", [False, True], ids=["max", "top2"])
@pytest.mark.parametrize("softmax", [False, True], ids=["sigmoid", "softmax"])
def test_groups(hip, E, groups, top_groups, K, top2, softmax):
    g = gen(E * groups + K)
    logits = torch.randn((19, E), device=DEV, generator=g) * 2
    bias = torch.randn((E,), device=DEV, generator=g) * 0.05
    check(hip, logits, bias, K, softmax=softmax, groups=groups, top_groups=top_groups, top2=top2)


@pytest.mark.parametrize("softmax", [False, True], ids=["sigmoid", "softmax"])
@pytest.mark.parametrize("groups,top_groups", [(1, 1), (8, 3)])
def test_ties_go_to_the_lower_index(hip, softmax, groups, top_groups):
    """Rows of few distinct logits, and all equal; bf16 makes them anyway."""
    g = gen(5)
    logits = torch.randint(0, 3, (40, 256), device=DEV, generator=g).float()
    logits[0] = 0.0
    logits[1] = -3.4028234663852886e38  # the type's lowest value: the score 0
    logits[1, 200:] = 1.0
    check(hip, logits, None, 16, softmax=softmax, groups=groups, top_groups=top_groups)
    check(hip, logits.bfloat16(), None, 16, softmax=softmax, groups=groups,
          top_groups=top_groups)


def test_minus_infinity_is_a_mask(hip):
    """Masked experts score 0; a row with fewer than K others takes masked
    ones of the lowest index last, with the weight 0."""
    logits = torch.full((3, 70), -math.inf, device=DEV)
    logits[0, 11], logits[0, 3], logits[1, 69] = 1.0, 2.0, 0.5
    logits[2] = 0.25
    for softmax in (False, True):
        check(hip, logits, None, 5, softmax=softmax)


@pytest.mark.parametrize("groups,top_groups", [(1, 1), (8, 3), (3, 2), (64, 5)])
def test_lowest_value_is_a_mask(hip, groups, top_groups):
    """Experts whose bias is the type's lowest value come after all others; a
    group of none but such (the sum of its two largest is minus infinity) last."""
    E = 192
    bias = torch.full((E,), torch.finfo(torch.float32).min, device=DEV)
    bias[5:9], bias[100], bias[150:153] = 0.25, 0.0, -1.0
    logits = torch.randn((5, E), device=DEV, generator=gen(12))
    for softmax in (False, True):
        for top2 in (False, True):
            check(hip, logits, bias, 6, softmax=softmax, groups=groups, top_groups=top_groups,
                  top2=top2)


def test_negative_bias_order(hip):
    """Adjusted scores below zero, and minus zero beside zero."""
    logits = torch.randn((9, 96), device=DEV, generator=gen(8))
    check(hip, logits, -torch.rand((96,), device=DEV, generator=gen(9)) - 1, 7)
    zero = torch.full((2, 96), -math.inf, device=DEV)
    zero[0, 50], zero[1, 7] = 0.0, 0.0
    bias = torch.zeros(96, device=DEV)
    bias[::2] = -0.0
    check(hip, zero, bias, 6)


def test_strided_rows(hip):
    wide = torch.randn((11, 500), device=DEV, generator=gen(3))
    check(hip, wide[:, 17:17 + 384], None, 16)
    check(hip, wide.bfloat16()[:, 3:3 + 101], None, 4, softmax=True)


@pytest.mark.parametrize("T", [2, 64])
@pytest.mark.parametrize("renorm", ["float", "double"])
def test_same_route_as_the_layer(hip, T, renorm):
    """The layer's own router on the layer's logits: ids and weights bit for bit."""
    k3x, ctx = hip
    H, I, E, K = 512, 256, 384, 16
    bank = k3x.Bank(ctx, k3x.LayerShape(H, I, E))
    bank.fill_synthetic(7, 119, 123)
    g = gen(T)
    bias = torch.randn((E,), device=DEV, generator=g) * 0.1
    bank.set_router_device(torch.randn((E, H), device=DEV, generator=g) * 0.05, bias,
                           torch.ones((H,), device=DEV))
    x = torch.randn((T, H), device=DEV, generator=g).bfloat16()
    taps = dict(logits=torch.empty((T, E), device=DEV),
                ids=torch.empty((T, K), dtype=torch.int32, device=DEV),
                weights=torch.empty((T, K), device=DEV))
    kind = k3x.RENORM_FLOAT if renorm == "float" else k3x.RENORM_DOUBLE
    p = k3x.make_params(T, K, 2.5, 1e-6, k3x.GLU_SWIGLU, 4.0, None, kind)
    k3x.check(k3x.moe_forward(ctx, bank, p, x, torch.empty_like(x), taps), "forward")
    st, ids, w = call(hip, taps["logits"], bias, K, renorm=renorm, scale=2.5)
    assert st == 0 and ctx.synchronize() == 0
    assert torch.equal(ids, taps["ids"]) and torch.equal(w, taps["weights"])
    bank.close()


@pytest.mark.parametrize("bad", [math.nan, math.inf])
@pytest.mark.parametrize("softmax", [False, True], ids=["sigmoid", "softmax"])
def test_bad_logits_are_latched(hip, bad, softmax):
    """The token's row stays as it was; the others' are written."""
    k3x, ctx = hip
    if bad == math.inf and not softmax:
        pytest.skip("a sigmoid of plus infinity is 1")
    logits = torch.randn((3, 384), device=DEV, generator=gen(1))
    logits[1, 77] = bad
    st, ids, w = call(hip, logits, None, 16, softmax=softmax)
    assert st == 0
    assert ctx.synchronize() == k3x.ERR_INVALID_STATE
    assert (ids[1] == -7).all() and (w[1] == -7).all()
    assert ctx.synchronize() == 0


def test_nothing_to_renormalise_is_latched(hip):
    k3x, ctx = hip
    logits = torch.full((1, 40), -math.inf, device=DEV)
    for renorm, code in (("float", k3x.ERR_INVALID_STATE), ("double", k3x.ERR_INVALID_EXTENT)):
        st, ids, _ = call(hip, logits, None, 4, renorm=renorm)
        assert st == 0 and ctx.synchronize() == code
        assert (ids == -7).all()
    st, ids, w = call(hip, logits, None, 4, renorm="none")
    assert st == 0 and ctx.synchronize() == 0
    assert ids.tolist() == [[0, 1, 2, 3]] and (w == 0).all()


def test_captured(hip):
    """Captured once, replayed on changed logits."""
    k3x, _ = hip
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        ctx = k3x.Context(0)
        own = (k3x, ctx)
        logits = torch.randn((37, 384), device=DEV, generator=gen(1))
        p = k3x.make_route_params(37, 384, 16)
        ids = torch.empty((37, 16), dtype=torch.int32, device=DEV)
        w = torch.empty((37, 16), device=DEV)
        graph = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, stream=s):
            assert k3x.route(ctx, p, logits, ids, w) == 0
        for i in range(3):
            logits.copy_(torch.randn((37, 384), device=DEV, generator=gen(10 + i)))
            graph.replay()
            got = ids.clone(), w.clone()
            st, ids2, w2 = call(own, logits, None, 16)
            assert st == 0 and ctx.synchronize() == 0
            assert torch.equal(got[0], ids2) and torch.equal(got[1], w2)
        ctx.close()


def test_logits_past_32_bits(hip):
    """2^32 logits, the most tokens and experts; the last tokens' routes."""
    k3x, ctx = hip
    T, E, K = 1 << 20, 4096, 4
    logits = torch.zeros((T, E), dtype=torch.bfloat16, device=DEV)
    logits[-3:] = torch.randn((3, E), device=DEV, generator=gen(77)).bfloat16()
    st, ids, w = call(hip, logits, None, K)
    assert st == 0 and ctx.synchronize() == 0
    want, weights = plain(logits[-3:], None, K)
    assert torch.equal(ids[-3:].cpu().long(), want)
    err = (w[-3:].cpu().double() - weights).abs()
    assert (err <= (4 + K) * 2.0 ** -24 * weights).all()
    assert torch.equal(ids[:-3].cpu(), torch.arange(K, dtype=torch.int32).expand(T - 3, K))
