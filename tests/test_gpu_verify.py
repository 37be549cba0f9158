"""Verification of drafted tokens (k3x_hip_verify_draft) against a plain
implementation in 64 bits, at the sizes, masks and borders where it can go
wrong.  Every output is a whole number and compared exactly: both sides form
probabilities and sums in double, so that they differ only where a uniform
falls within about 1e-12 of a border, which the drawn uniforms (multiples of
2^-24) do not."""
from __future__ import annotations

import math

import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")
DEV = "cuda:0"
F32, BF16 = torch.float32, torch.bfloat16


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


def inputs(N, D, V, dtype=F32, probs=False, dist=True, seed=0, close=0.8):
    g = gen(seed + N * 1000 + D * 100 + V)
    target = torch.randn((N, D + 1, V), device=DEV, generator=g) * 2
    draft = target[:, :D] + torch.randn((N, D, V), device=DEV, generator=g) * close
    s = dict(tokens=torch.distributions.Categorical(logits=draft).sample().to(torch.int32)
             if D and dist else draft.argmax(-1).to(torch.int32) if D
             else torch.empty((N, 0), dtype=torch.int32, device=DEV))
    if probs:
        target, draft = target.softmax(-1), draft.softmax(-1)
    s["target"], s["draft"] = target.to(dtype), draft.to(dtype) if dist else None
    s["accept_u"] = torch.rand((N, D), device=DEV, generator=g)
    s["sample_u"] = torch.rand((N,), device=DEV, generator=g)
    return s


def definition(s, probs, greedy, temperature, counts=None):
    N, D1, V = s["target"].shape
    accepted, out = torch.zeros(N, dtype=torch.int32), torch.full((N, D1), -1, dtype=torch.int32)
    temperature = float(torch.tensor(temperature))

    def dist(row):
        row = row.double().cpu()
        return row if probs else torch.softmax(row / temperature, 0)

    for n in range(N):
        D = D1 - 1 if counts is None else counts[n]
        if D == -1:
            continue
        i = 0
        while i < D:
            x = int(s["tokens"][n, i])
            if greedy:
                row = s["target"][n, i].float()
                if int((row == row.max()).nonzero()[0]) != x:
                    break
            else:
                q = 1.0 if s["draft"] is None else float(dist(s["draft"][n, i])[x])
                if not float(s["accept_u"][n, i]) * q < float(dist(s["target"][n, i])[x]):
                    break
            out[n, i] = x
            i += 1
        accepted[n] = i
        if greedy:
            row = s["target"][n, i].float()
            out[n, i] = int((row == row.max()).nonzero()[0])
            continue
        p = dist(s["target"][n, i])
        rest = p.clone()
        if i < D and s["draft"] is None:
            rest[int(s["tokens"][n, i])] = 0
        elif i < D:
            rest = (rest - dist(s["draft"][n, i])).clamp(min=0)
        if not float(rest.sum()) > 0:
            rest = p
        cum = rest.cumsum(0)
        out[n, i] = int((cum > float(s["sample_u"][n]) * cum[-1]).nonzero()[0])
    return accepted, out


def call(hip, s, probs=False, greedy=False, temperature=1.0, counts=None):
    k3x, ctx = hip
    N, D1, V = s["target"].shape
    p = k3x.make_verify_params(s["target"], k3x.DIST_PROBS if probs else k3x.DIST_LOGITS, greedy,
                               temperature)
    accepted = torch.full((N,), -7, dtype=torch.int32, device=DEV)
    out = torch.full((N, D1), -7, dtype=torch.int32, device=DEV)
    ws = torch.empty((k3x.verify_workspace_bytes(p),), dtype=torch.uint8, device=DEV)
    c = None if counts is None else torch.tensor(counts, dtype=torch.int32, device=DEV)
    st = k3x.verify_draft(ctx, p, s["target"], s["tokens"], accepted, out, draft=s["draft"],
                          draft_counts=c, accept_u=None if greedy else s["accept_u"],
                          sample_u=None if greedy else s["sample_u"], workspace=ws)
    return st, accepted, out


def check(hip, s, probs=False, greedy=False, temperature=1.0, counts=None):
    k3x, ctx = hip
    print(f"[gpu-test] verify {tuple(s['target'].shape)} {s['target'].dtype} probs={probs} "
          f"greedy={greedy} draft={s['draft'] is not None} counts={counts}", flush=True)
    st, accepted, out = call(hip, s, probs, greedy, temperature, counts)
    assert st == 0
    assert ctx.synchronize() == 0
    want_a, want = definition(s, probs, greedy, temperature, counts)
    assert torch.equal(accepted.cpu(), want_a)
    assert torch.equal(out.cpu(), want)
    return want_a


@pytest.mark.parametrize("N,D,V", [(1, 1, 1), (1, 0, 7), (2, 3, 2), (5, 4, 63), (3, 2, 64),
                                   (2, 64, 65), (9, 5, 257), (4, 7, 4096), (3, 4, 4097),
                                   (2, 2, 32003), (1, 3, 163840), (1, 1, 300001)])
@pytest.mark.parametrize("dtype", [F32, BF16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("probs", [False, True], ids=["logits", "probs"])
@pytest.mark.parametrize("dist", [False, True], ids=["one_hot", "draft"])
def test_sampled(hip, N, D, V, dtype, probs, dist):
    check(hip, inputs(N, D, V, dtype, probs, dist), probs, temperature=1.0 if probs else 0.7)


@pytest.mark.parametrize("N,D,V", [(1, 1, 1), (1, 0, 7), (6, 4, 63), (2, 64, 130), (4, 7, 4097),
                                   (2, 3, 163840)])
@pytest.mark.parametrize("dtype", [F32, BF16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("probs", [False, True], ids=["logits", "probs"])
def test_greedy(hip, N, D, V, dtype, probs):
    check(hip, inputs(N, D, V, dtype, probs, False, close=0.05), probs, greedy=True)


def test_greedy_ties_go_to_the_lower_token(hip):
    s = inputs(4, 3, 9000, dist=False)
    s["target"] = torch.randint(0, 2, s["target"].shape, device=DEV, generator=gen(2)).float()
    s["target"][0] = 0
    s["tokens"][:] = s["target"][:, :3].argmax(-1)
    s["tokens"][0] = 0
    check(hip, s, greedy=True)


@pytest.mark.parametrize("probs", [False, True], ids=["logits", "probs"])
def test_counts_and_skipped_sequences(hip, probs):
    """Fewer drafts, none, and sequences left out, whose rows may hold anything."""
    s = inputs(6, 5, 1000, probs=probs)
    s["target"][2] = math.nan
    s["draft"][2] = math.nan
    s["target"][1, 3:] = math.nan
    s["draft"][1, 2:] = math.nan
    s["tokens"][1, 2:] = -1
    check(hip, s, probs, counts=[5, 2, -1, 0, 1, 3])
    s["draft"] = None
    check(hip, s, probs, counts=[5, 2, -1, 0, 1, 3])


def test_masked_tokens(hip):
    """Minus infinity is a token that never comes; the type's lowest value too."""
    s = inputs(8, 4, 5000)
    mask = torch.rand(s["target"].shape, device=DEV, generator=gen(1)) < 0.9
    s["target"] = s["target"].masked_fill(mask, -math.inf)
    s["draft"] = s["draft"].masked_fill(mask[:, :4], torch.finfo(F32).min)
    s["tokens"] = s["draft"].argmax(-1).to(torch.int32)
    check(hip, s)
    only = inputs(3, 2, 5000)
    only["target"][:] = -math.inf
    only["target"][:, :, 4321] = -3.0
    check(hip, only)
    s["draft"][:, :, 17] = math.inf  # in rows that a one-hot call does not read
    s["draft"] = None
    check(hip, s)


@pytest.mark.parametrize("probs", [False, True], ids=["logits", "probs"])
def test_equal_distributions_are_accepted(hip, probs):
    s = inputs(7, 5, 3000, probs=probs)
    s["draft"] = s["target"][:, :5].clone()
    s["accept_u"][:] = 1 - 2.0 ** -24
    assert (check(hip, s, probs) == 5).all()


def test_nothing_left_over_the_draft(hip):
    """Probabilities of a draft that covers the target's: drawn from the target's."""
    s = inputs(5, 1, 3000, probs=True)
    s["draft"] = s["target"][:, :1] * 2
    s["accept_u"][:] = 0.75
    assert (check(hip, s, True) == 0).all()
    one = inputs(2, 1, 600, probs=True, dist=False)  # the drafted token was all there was
    one["target"][:] = 0
    one["target"][:, :, 599] = 0.5
    one["tokens"][:] = 599
    one["accept_u"][:] = 0.9
    assert (check(hip, one, True) == 0).all()


@pytest.mark.parametrize("u", [0.0, 2.0 ** -149, 0.5, 1 - 2.0 ** -24])
def test_borders_of_the_uniforms(hip, u):
    """First and last token over 0, flat probabilities, borders that are exact."""
    s = inputs(4, 2, 8192, probs=True)
    s["target"][:] = 1 / 8192
    s["target"][:, :, :5] = 0
    s["target"][:, :, -7:] = 0
    s["draft"][:] = 1 / 4096
    s["accept_u"][:] = u
    s["sample_u"][:] = u
    check(hip, s, True)
    s["draft"] = None
    check(hip, s, True)


def test_large_logits(hip):
    s = inputs(3, 3, 2000)
    for x in ("target", "draft"):
        s[x] = s[x] * 1e4 + 3e37
    check(hip, s)
    s = inputs(3, 3, 2000)
    check(hip, s, temperature=1e-3)
    check(hip, s, temperature=1e3)


@pytest.mark.parametrize("fault", ["nan", "inf", "token", "uniform", "sample", "empty", "count",
                                   "draft"])
def test_faults_are_latched(hip, fault):
    """The sequence's outputs stay as they were, the others' are written or left."""
    k3x, ctx = hip
    s = inputs(3, 3, 700)
    s["accept_u"][:] = 0
    counts = None
    if fault in ("nan", "inf"):
        s["target"][1, 1, 650] = math.nan if fault == "nan" else math.inf
    elif fault == "token":
        s["tokens"][1, 0] = 700
    elif fault == "uniform":
        s["accept_u"][1, 0] = 1.0
    elif fault == "sample":
        s["sample_u"][1] = -0.5
    elif fault == "empty":
        s["target"][1, 0] = -math.inf
    elif fault == "draft":
        s["draft"][1, 0, 3] = math.nan
    else:
        counts = [3, 4, 3]
    st, accepted, out = call(hip, s, counts=counts)
    assert st == 0 and ctx.synchronize() == k3x.ERR_INVALID_STATE
    assert accepted[1] == -7 and (out[1] == -7).all()
    check(hip, inputs(3, 3, 700))


@pytest.mark.parametrize("bad", [-1e-3, math.nan, math.inf])
def test_bad_probabilities_are_latched(hip, bad):
    k3x, ctx = hip
    for which in ("target", "draft"):
        s = inputs(2, 1, 900, probs=True)
        s["accept_u"][:] = 1 - 2.0 ** -24
        s["draft"][1, 0, int(s["tokens"][1, 0])] = 0.99  # not accepted
        at = (int(s["tokens"][1, 0]) + 5) % 900
        s[which][1, 0, at] = bad
        st, accepted, out = call(hip, s, True)
        assert st == 0 and ctx.synchronize() == k3x.ERR_INVALID_STATE
        assert accepted[1] == -7


def test_captured(hip):
    """Captured once; replays on changed rows equal eager calls."""
    k3x, _ = hip
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        ctx = k3x.Context(0)
        s = inputs(5, 4, 20000)
        p = k3x.make_verify_params(s["target"], temperature=0.9)
        ws = torch.zeros((k3x.verify_workspace_bytes(p),), dtype=torch.uint8, device=DEV)
        accepted = torch.zeros((5,), dtype=torch.int32, device=DEV)
        out = torch.zeros((5, 5), dtype=torch.int32, device=DEV)
        graph = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, stream=stream):
            assert k3x.verify_draft(ctx, p, s["target"], s["tokens"], accepted, out,
                                    draft=s["draft"], accept_u=s["accept_u"],
                                    sample_u=s["sample_u"], workspace=ws) == 0
        for i in range(3):
            new = inputs(5, 4, 20000, seed=i + 1)
            for x in s:
                s[x].copy_(new[x])
            graph.replay()
            got = accepted.clone(), out.clone()
            st, a2, o2 = call((k3x, ctx), s, temperature=0.9)
            assert st == 0 and ctx.synchronize() == 0
            assert torch.equal(got[0], a2) and torch.equal(got[1], o2)
        ctx.close()


@pytest.mark.parametrize("greedy", [True, False], ids=["greedy", "sampled"])
def test_rows_past_32_bits(hip, greedy):
    """2^32 entries and more of the longest rows; the last sequence's tokens."""
    k3x, ctx = hip
    N, D, V = 1366, 2, 1 << 20
    s = dict(target=torch.zeros((N, D + 1, V), dtype=BF16, device=DEV), draft=None,
             tokens=torch.zeros((N, D), dtype=torch.int32, device=DEV))
    g = gen(5)
    s["target"][-1].copy_(torch.randn((D + 1, V), device=DEV, generator=g) * 3)
    s["tokens"][-1, 0] = s["target"][-1, 0].float().argmax()
    s["accept_u"] = torch.full((N, D), 2.0 ** -30, device=DEV)
    s["sample_u"] = torch.rand((N,), device=DEV, generator=g)
    st, accepted, out = call(hip, s, greedy=greedy)
    assert st == 0 and ctx.synchronize() == 0
    last = {x: None if y is None else y[-1:] for x, y in s.items()}
    want_a, want = definition(last, False, greedy, 1.0)
    assert torch.equal(accepted[-1:].cpu(), want_a) and torch.equal(out[-1:].cpu(), want)
    if greedy:  # rows of equal entries: the lowest token
        assert (accepted[:-1] == D).all() and (out[:-1] == 0).all()


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("probs", [False, True], ids=["logits", "probs"])
@pytest.mark.parametrize("greedy", [False, True], ids=["sampled", "greedy"])
@pytest.mark.parametrize("pad", [3, 64])
def test_padded_rows(hip, dtype, probs, greedy, pad):
    """Rows of a padded vocabulary as they lie: what the padding holds is not looked at."""
    s = inputs(3, 2, 2049, dtype, probs)
    for x in ("target", "draft"):
        rows = torch.full((*s[x].shape[:2], 2049 + pad), math.nan, device=DEV).to(dtype)
        rows[..., :2049] = s[x]
        s[x] = rows[..., :2049]
    check(hip, s, probs, greedy)


def test_entries_that_are_not_used(hip):
    """Probabilities of accepted rows are looked at for the drafted token only, rows past the
    first draft that is not accepted not at all."""
    s = inputs(2, 4, 3000, probs=True)
    s["accept_u"][:] = 0
    s["accept_u"][:, 2] = 1 - 2.0 ** -24
    at = torch.arange(2, device=DEV)
    x = s["tokens"][:, 2].long()
    s["draft"][at, 2, x], s["target"][at, 2, x] = 1.0, 1e-9  # not accepted
    clean = {k: v.clone() for k, v in s.items()}
    for i in range(2):
        for name in ("target", "draft"):
            keep = s[name][at, i, s["tokens"][:, i].long()].clone()
            s[name][:, i] = math.nan
            s[name][at, i, s["tokens"][:, i].long()] = keep
    s["target"][:, 3:] = math.inf
    s["draft"][:, 3:] = -1.0
    s["tokens"][:, 3] = -1
    k3x, ctx = hip
    assert (check(hip, clean, True) == 2).all()
    st, accepted, out = call(hip, s, True)
    st2, accepted2, out2 = call(hip, clean, True)
    assert st == st2 == 0 and ctx.synchronize() == 0
    assert torch.equal(accepted, accepted2) and torch.equal(out, out2)
