"""Penalties, biases and masks on logits (k3x_hip_adjust_logits) against a plain implementation.

The kernel's steps are fp32 operations in a given order, each rounded once, and so are the plain
form's here, in the same order: outputs are compared bit by bit (NaN as NaN).  Against 64 bits each
of the five operations is off by half a step of fp32 of its result, the last rounding by half a
step of the type."""
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
    g = torch.Generator()
    g.manual_seed(seed)
    return g


def make(N, D, V, dtype=F32, width=50, biases=7, masks=3, seed=0):
    """Inputs on the host."""
    g = gen(seed + 1000 * N + 10 * D + V)
    s = dict(logits=(torch.randn((N, D + 1, V), generator=g) * 3).to(dtype))
    lens = torch.randint(0, width + 1, (N,), generator=g)
    s["history"] = torch.randint(0, min(V, 40), (N, width), generator=g).int()
    far = torch.rand((N, width), generator=g) < 0.5
    s["history"][far] = torch.randint(0, V, (int(far.sum()),), generator=g).int()
    s["history_lens"] = lens.int()
    s["prompt_lens"] = (lens * torch.rand(N, generator=g)).int()
    s["drafts"] = torch.randint(0, min(V, 60), (N, D), generator=g).int()
    s["repetition"] = 0.6 + torch.rand(N, generator=g)
    s["frequency"] = torch.rand(N, generator=g) - 0.3
    s["presence"] = torch.rand(N, generator=g) - 0.3
    if biases:
        counts = torch.randint(0, 2 * biases, (N,), generator=g)
        offsets = torch.cat([counts.new_zeros(1), counts.cumsum(0)]).int()
        n = int(offsets[-1])
        s["bias"] = (offsets, torch.randint(0, V, (n,), generator=g).int(),
                     torch.randn(n, generator=g) * 5)
    if masks:
        s["masks"] = torch.randint(-1 << 31, 1 << 31, (masks, -(-V // 32)),
                                   generator=g).int()
        s["mask_index"] = torch.randint(-1, masks, (N, D + 1), generator=g).int()
    return s


def definition(s, counts=None, wide=False):
    """Row by row in fp32 (wide: in 64 bits, and the tolerance); rows left out are NaN."""
    x = s["logits"]
    N, D1, V = x.shape
    real = torch.float64 if wide else F32
    want = torch.full(x.shape, math.nan, dtype=torch.float64)
    tol = torch.zeros(x.shape, dtype=torch.float64)
    for n in range(N):
        D = D1 - 1 if counts is None else counts[n]
        if D == -1:
            continue
        seen = torch.zeros(V, dtype=torch.bool)
        times = torch.zeros(V)
        if s.get("history") is not None:
            total = int(s["history_lens"][n])
            prompt = int(s["prompt_lens"][n]) if s.get("prompt_lens") is not None else 0
            h = s["history"][n].long()
            seen[h[:total]] = True
            times += torch.bincount(h[prompt:total], minlength=V)
        bias, has = torch.zeros(V, dtype=real), torch.zeros(V, dtype=torch.bool)
        if s.get("bias") is not None:
            o, t, v = s["bias"]
            for i in range(int(o[n]), int(o[n + 1])):
                bias[t[i]], has[t[i]] = v[i].to(real), True
        for r in range(D + 1):
            l = x[n, r].to(real)
            off = torch.zeros(V, dtype=torch.float64)

            def step(y, where):
                off.add_(torch.where(where, y.double().abs() * 2.0 ** -24, 0.0))
                return torch.where(where, y, l)
            if s.get("repetition") is not None:
                p = s["repetition"][n].to(real)
                l = step(torch.where(l > 0, l / p, l * p), seen)
            if s.get("frequency") is not None:
                c = (s["frequency"][n].to(real) * times.to(real))
                off.add_(c.double().abs() * 2.0 ** -24)
                l = step(l - c, times > 0)
            if s.get("presence") is not None:
                l = step(l - s["presence"][n].to(real), times > 0)
            if s.get("bias") is not None:
                l = step(l + bias, has)
            if s.get("masks") is not None and int(s["mask_index"][n, r]) >= 0:
                w = s["masks"][int(s["mask_index"][n, r])].long()
                bits = (w[:, None] >> torch.arange(32)) & 1
                l = torch.where(bits.reshape(-1)[:V].bool(), l, -math.inf)
            if wide:
                half = 2.0 ** (-24 if x.dtype == F32 else -8)
                tol[n, r] = off * (1 + half) + l.abs() * half
                want[n, r] = l
            else:
                want[n, r] = l.to(x.dtype).double()
            if r < D:
                t = int(s["drafts"][n, r])
                seen[t] = True
                times[t] += 1
    return (want, tol) if wide else want


def call(hip, s, counts=None, in_place=False, pad=0, **kw):
    k3x, ctx = hip
    d = {k: tuple(t.to(DEV) for t in v) if isinstance(v, tuple) else v.to(DEV)
         for k, v in s.items() if v is not None}
    x = d.pop("logits")
    N, D1, V = x.shape
    if pad:
        wide = torch.full((N, D1, V + pad), 5.0, dtype=x.dtype, device=DEV)
        wide[..., :V] = x
        x = wide[..., :V]
    out = x if in_place else torch.full_like(x, 7.0, memory_format=torch.contiguous_format)
    if counts is not None:
        d["draft_counts"] = torch.tensor(counts, dtype=torch.int32, device=DEV)
    d.update(kw)
    st = k3x.adjust_logits(ctx, k3x.make_logits_params(x), x, out, **d)
    return st, out, x


def check(hip, s, counts=None, **kw):
    k3x, ctx = hip
    print(f"[gpu-test] logits {tuple(s['logits'].shape)} {s['logits'].dtype} "
          f"{sorted(k for k in s if s[k] is not None)} counts={counts} {kw}", flush=True)
    st, out, x = call(hip, s, counts, **kw)
    assert (st, ctx.synchronize()) == (0, 0)
    want = definition(s, counts)
    left = torch.isnan(want) & ~torch.isnan(s["logits"].double())
    got = out.double().cpu()
    rows = left.all(-1)
    if counts is not None:  # rows that are left as they were
        assert torch.equal(got[rows], s["logits"][rows].double() if kw.get("in_place")
                           else torch.full_like(got[rows], 7.0))
    a, b = got[~rows], want[~rows]
    assert torch.equal(torch.isnan(a), torch.isnan(b))
    assert torch.equal(a.nan_to_num(123.0), b.nan_to_num(123.0))
    if kw.get("pad") and kw.get("in_place"):
        assert (out.as_strided((out.shape[0], out.shape[1], kw["pad"]), out.stride(),
                               out.shape[2]) == 5).all()


@pytest.mark.parametrize("N,D,V", [(1, 0, 1), (1, 1, 31), (2, 3, 32), (3, 4, 33), (2, 2, 1000),
                                   (5, 4, 4095), (1, 7, 4096), (2, 1, 4097), (3, 3, 20011),
                                   (1, 64, 130), (1, 2, 300001)])
@pytest.mark.parametrize("dtype", [F32, BF16], ids=["fp32", "bf16"])
def test_all_steps(hip, N, D, V, dtype):
    check(hip, make(N, D, V, dtype))


@pytest.mark.parametrize("V", [1000, 5001])
def test_against_64_bits(hip, V):
    for dtype in (F32, BF16):
        s = make(4, 3, V, dtype)
        st, out, _ = call(hip, s)
        assert (st, hip[1].synchronize()) == (0, 0)
        want, tol = definition(s, wide=True)
        got = out.double().cpu()
        fine = torch.isfinite(want)
        assert torch.equal(got[~fine], want[~fine])
        assert ((got - want).abs()[fine] <= tol[fine]).all()


STEPS = ["repetition", "frequency", "presence", "bias", "masks", "history"]


@pytest.mark.parametrize("only", STEPS)
@pytest.mark.parametrize("without", [False, True], ids=["only", "without"])
def test_single_steps(hip, only, without):
    s = make(3, 2, 5000)
    for k in STEPS:
        if (k == only) == without:
            s[k] = None
            if k == "masks":
                s["mask_index"] = None
            if k == "history":
                s["history_lens"] = s["prompt_lens"] = None
    check(hip, s)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("pad", [0, 1, 7, 8])
def test_in_place_and_padded_rows(hip, dtype, pad):
    check(hip, make(3, 2, 4321, dtype), in_place=True, pad=pad)
    check(hip, make(3, 2, 4321, dtype), pad=pad)


@pytest.mark.parametrize("in_place", [False, True], ids=["out", "in_place"])
def test_counts_and_skipped_sequences(hip, in_place):
    s = make(6, 5, 1000)
    s["drafts"][1, 2:] = -1  # not reached
    s["history_lens"][2] = 9999
    s["repetition"][2] = math.nan
    s["mask_index"][2] = 77
    check(hip, s, counts=[5, 2, -1, 0, 1, 3], in_place=in_place)


def test_history_of_every_kind(hip):
    """Empty, all prompt, all answer, one token many times, at the parts' borders."""
    s = make(5, 3, 9000, width=3000)
    s["history_lens"] = torch.tensor([0, 3000, 3000, 3000, 1]).int()
    s["prompt_lens"] = torch.tensor([0, 3000, 0, 1500, 1]).int()
    s["history"][3] = 4096
    s["history"][2, ::2] = 4095
    s["drafts"][0] = torch.tensor([8999, 8999, 0])
    check(hip, s)
    s["prompt_lens"] = None
    check(hip, s)


def test_rows_of_masks_and_histories_apart(hip):
    k3x, ctx = hip
    s = make(3, 1, 2000)
    wide = torch.zeros((3, 63 + 5), dtype=torch.int32)
    wide[:, :63] = s["masks"]
    st, out, _ = call(hip, s, masks=wide.to(DEV)[:, :63])
    assert (st, ctx.synchronize()) == (0, 0)
    assert torch.equal(out.double().cpu(), definition(s))


def test_values_go_through(hip):
    """Infinities, NaN and the type's lowest value among logits and biases."""
    s = make(2, 2, 3000)
    for i, v in enumerate([math.inf, -math.inf, math.nan, torch.finfo(F32).min,
                           torch.finfo(F32).max, 0.0, -0.0, 1e-40]):
        s["logits"][:, :, i::40] = v
    o, t, v = s["bias"]
    v[0], v[1] = -math.inf, math.inf
    check(hip, s)
    s["masks"][:] = 0  # nothing is allowed
    check(hip, s)


def test_of_several_biases_the_last_holds(hip):
    s = make(2, 1, 5000)
    s["bias"] = (torch.tensor([0, 300, 301]).int(), torch.full((301,), 4097).int(),
                 torch.arange(301).float())
    check(hip, s)


@pytest.mark.parametrize("what", ["history", "prompt", "token", "draft", "bias", "bias offsets",
                                  "mask", "count", "repetition", "zero", "frequency", "presence"])
def test_unfit_sequences_are_latched(hip, what):
    k3x, ctx = hip
    s = make(3, 2, 1000, biases=4)
    s["bias"] = (torch.tensor([0, 2, 4, 6]).int(), torch.arange(6).int(), torch.ones(6))
    counts = None
    s["history_lens"][1], s["prompt_lens"][1] = 20, 10
    if what == "history":
        s["history_lens"][1] = 51
    elif what == "prompt":
        s["prompt_lens"][1] = 21
    elif what == "token":
        s["history"][1, 7] = 1000
    elif what == "draft":
        s["drafts"][1, 1] = 1000
    elif what == "bias":
        s["bias"][1][3] = 1000
    elif what == "bias offsets":
        s["bias"][0][2] = 1
    elif what == "mask":
        s["mask_index"][1, 0] = 3
    elif what == "count":
        counts = [2, 3, 2]
    elif what == "zero":
        s["repetition"][1] = 0.0
    else:
        s[what][1] = math.nan
    print(f"[gpu-test] logits with unfit {what}", flush=True)
    st, out, _ = call(hip, s, counts)
    assert (st, ctx.synchronize()) == (0, k3x.ERR_INVALID_STATE)
    assert ctx.synchronize() == 0


def test_capture_and_replay(hip):
    """Replays read what the buffers hold then."""
    k3x, ctx0 = hip
    s = make(4, 3, 20011, BF16)
    d = {k: tuple(t.to(DEV) for t in v) if isinstance(v, tuple) else v.to(DEV)
         for k, v in s.items()}
    x = d.pop("logits")
    out = torch.zeros_like(x)
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        ctx = k3x.Context(0)
        p = k3x.make_logits_params(x)
        assert k3x.adjust_logits(ctx, p, x, out, **d) == 0
        assert ctx.synchronize() == 0
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            assert k3x.adjust_logits(ctx, p, x, out, **d) == 0
    for i in range(4):
        t = make(4, 3, 20011, BF16, seed=i)
        t["bias"] = s["bias"]
        for k, v in t.items():
            if k == "logits":
                x.copy_(v)
            elif k != "bias":
                d[k].copy_(v)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert ctx.synchronize() == 0
        want = definition(t)
        assert torch.equal(out.double().cpu(), want)
    ctx.close()
