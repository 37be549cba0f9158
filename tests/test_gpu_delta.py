"""The gated delta rule (k3x_hip_delta_rule) against its definition in 64
bits, token by token, at the lengths, shapes, gates and offsets where it can go
wrong.

Bound.  Take one value column s of a head's state, M the largest 2-norm that it
and the values take.  A token's exact update s -> (I - beta k k^T) D s + beta v k
does not lengthen an error (|k| <= 1, 0 <= beta <= 1, 0 <= D <= 1), so errors
only add up over a sequence's L tokens, and those of one token are, in units of
2^-24 M: the decay's exponential and product 4, the normalised key 6 in each of
its two uses, the dot product over K (lane sums of 16 and four levels, or chunk
sums of 32 over halves of 11 bits each, whose products leave 2^-22 each) 24, the
update 4, the chunk's inverse another 24: below 96 together.  Hence
|error| <= 96 L 2^-24 M for the state, times scale |q| for an output, plus half a
step of the output's type."""
from __future__ import annotations

import math

import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")
DEV = "cuda:0"
EPS = 1e-6
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


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


def inputs(lens, Hk, H, K, V, dtype=F32, gate="channel", seed=0, extra=0, strong=1.0):
    """Inputs of sequences of these lengths, `extra` rows behind the last."""
    g = gen(seed + 1000 * sum(lens) + K)
    T = sum(lens) + extra

    def n(*shape):
        return torch.randn(shape, device=DEV, generator=g)

    s = dict(lens=list(lens), q=n(T, Hk, K).to(dtype), k=n(T, Hk, K).to(dtype),
             v=n(T, H, V).to(dtype), beta=torch.sigmoid(n(T, H)), gate=None,
             state=n(len(lens), H, K, V) * 0.3)
    if gate != "none":
        s["gate"] = -strong * torch.nn.functional.softplus(
            n(T, H, K) * 2 - 3 if gate == "channel" else n(T, H) * 2 - 3)
    cu = [0]
    for x in lens:
        cu.append(cu[-1] + x)
    s["offsets"] = torch.tensor(cu, dtype=torch.int32, device=DEV)
    return s


def definition(s, scale, norm=True, limits=None, state=True):
    """out, states and their bounds, in 64 bits."""
    q, k, v = (s[x].double() for x in "qkv")
    H, K, V = v.shape[1], q.shape[2], v.shape[2]
    r = H // q.shape[1]
    if norm:
        q = q / (q.square().sum(-1, keepdim=True) + EPS).sqrt()
        k = k / (k.square().sum(-1, keepdim=True) + EPS).sqrt()
    q, k = q.repeat_interleave(r, 1), k.repeat_interleave(r, 1)
    S = s["state"].double().clone() if state else torch.zeros_like(s["state"]).double()
    out, tol = torch.zeros_like(v), torch.zeros_like(v)
    stol = torch.zeros_like(S)
    at = 0
    for n, length in enumerate(s["lens"]):
        most = length if limits is None else min(length, limits[n])
        M = S[n].square().sum(1).sqrt()  # [H][V]
        for i in range(most):
            t = at + i
            if s["gate"] is not None:
                d = s["gate"][t].double().exp()
                S[n] *= d[..., None] if d.dim() == 2 else d[:, None, None]
            u = s["beta"][t].double()[:, None] * (v[t] - (S[n] * k[t][..., None]).sum(1))
            S[n] += k[t][..., None] * u[:, None]
            out[t] = scale * (S[n] * q[t][..., None]).sum(1)
            M = torch.maximum(torch.maximum(M, S[n].square().sum(1).sqrt()), v[t].abs())
            tol[t] = 96 * (i + 1) * 2.0 ** -24 * M * scale * q[t].square().sum(-1).sqrt()[:, None]
        stol[n] = (96 * most * 2.0 ** -24 * M)[:, None]
        at += length
    return out, S, tol, stol


def call(hip, s, scale=None, norm=True, limits=None, slot_index=None, state_in="own",
         state_out="new", slots=None, out=None, offsets="own", longest=None):
    k3x, ctx = hip
    scale = s["q"].shape[-1] ** -0.5 if scale is None else scale
    state_in = s["state"] if isinstance(state_in, str) else state_in
    N = len(s["lens"])
    if isinstance(state_out, str):
        state_out = torch.full_like(s["state"], -7.0)
    p = k3x.make_delta_params(s["q"], s["k"], s["v"], N, gate=s["gate"], scale=scale,
                              norm_epsilon=EPS if norm else 0.0,
                              longest=max(s["lens"]) if longest is None else longest, slots=slots)
    out = torch.full(s["v"].shape, -7.0, device=DEV).to(s["v"].dtype) if out is None else out
    need = k3x.delta_workspace_bytes(p)
    ws = torch.empty((need,), dtype=torch.uint8, device=DEV) if need else None
    lim = None if limits is None else torch.tensor(limits, dtype=torch.int32, device=DEV)
    st = k3x.delta_rule(ctx, p, s["q"], s["k"], s["v"], s["beta"], out, gate=s["gate"],
                        offsets=s["offsets"] if isinstance(offsets, str) else offsets, limits=lim,
                        slot_index=slot_index, state_in=state_in, state_out=state_out,
                        workspace=ws)
    return st, out, state_out


def close(got, want, tol, dtype=F32):
    step = 0.0 if dtype == F32 else torch.finfo(dtype).eps / 2
    err = (got.double() - want).abs()
    worst = float((err / (tol + 2.0 ** -24 * want.abs() + step * want.abs() + 1e-30)).max()) \
        if err.numel() else 0.0
    assert worst <= 1.0, worst
    return worst


def check(hip, s, parity_report=None, **kw):
    k3x, ctx = hip
    lens = s["lens"]
    print(f"[gpu-test] delta {lens} q{tuple(s['q'].shape)} v{tuple(s['v'].shape)} {s['v'].dtype}"
          f" gate {None if s['gate'] is None else s['gate'].dim()} {sorted(kw)}", flush=True)
    scale = kw.get("scale", s["q"].shape[-1] ** -0.5)
    st, out, state = call(hip, s, **kw)
    assert st == 0
    assert ctx.synchronize() == 0
    want, S, tol, stol = definition(s, scale, kw.get("norm", True), kw.get("limits"),
                                    isinstance(kw.get("state_in", "own"), str))
    live = torch.zeros(len(out), dtype=torch.bool, device=DEV)
    at = 0
    for n, length in enumerate(lens):
        live[at:at + min(length, (kw.get("limits") or {n: length})[n])] = True
        at += length
    a = close(out[live], want[live], tol[live], s["v"].dtype)
    b = close(state, S, stol) if state is not None else 0.0
    assert (out[~live] == -7).all()
    if parity_report:
        parity_report(f"out at {a:.3f} and state at {b:.3f} of the bound")
    return out, state


SHAPES = [(1, 1, 1, 1), (1, 1, 16, 16), (2, 2, 33, 47), (1, 4, 64, 64), (2, 2, 96, 80),
          (2, 4, 128, 128), (1, 2, 128, 20), (1, 1, 129, 33), (1, 2, 256, 64), (1, 1, 8, 200)]


@pytest.mark.parametrize("Hk,H,K,V", SHAPES)
@pytest.mark.parametrize("gate", ["none", "head", "channel"])
@pytest.mark.parametrize("lens", [(1,), (1, 1, 1), (0, 3, 17), (70, 0, 1, 33)],
                         ids=lambda x: "_".join(map(str, x)))
def test_shapes(hip, Hk, H, K, V, gate, lens):
    check(hip, inputs(lens, Hk, H, K, V, gate=gate))


@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("gate", ["none", "head", "channel"])
@pytest.mark.parametrize("lens", [(1, 1), (5, 16, 2), (40, 31, 32, 64, 65), (300, 129)],
                         ids=lambda x: "_".join(map(str, x)))
def test_types(hip, dtype, gate, lens, parity_report):
    check(hip, inputs(lens, 2, 4, 128, 128, dtype, gate), parity_report)


@pytest.mark.parametrize("length", [1, 2, 15, 16, 17, 31, 32, 33, 47, 48, 49, 63, 64, 65, 127, 128,
                                    129, 200])
@pytest.mark.parametrize("gate", ["head", "channel"])
def test_lengths(hip, length, gate):
    check(hip, inputs((length,), 1, 1, 64, 32, BF16, gate))


@pytest.mark.parametrize("strong", [0.0, 1e-4, 30.0, 300.0])
@pytest.mark.parametrize("gate", ["head", "channel"])
@pytest.mark.parametrize("lens", [(3,), (150,)], ids=["short", "long"])
def test_decays(hip, strong, gate, lens):
    """No decay at all, next to none, and decays past every exponent."""
    check(hip, inputs(lens, 1, 2, 128, 64, gate=gate, strong=strong))


@pytest.mark.parametrize("gate", ["head", "channel"])
@pytest.mark.parametrize("lens", [(6,), (100,)], ids=["short", "long"])
def test_minus_infinity_empties_the_state(hip, gate, lens):
    s = inputs(lens, 1, 2, 64, 32, gate=gate)
    s["gate"][4] = -math.inf
    s["gate"][lens[0] // 2, 0] = -math.inf
    check(hip, s)


@pytest.mark.parametrize("lens", [(7,), (90,)], ids=["short", "long"])
@pytest.mark.parametrize("size", [1e-18, 1e-3, 30.0, 1e15])
def test_sizes_of_values(hip, lens, size):
    """The state is linear in the values, whatever their size."""
    s = inputs(lens, 1, 1, 128, 48)
    s["v"] *= size
    s["state"] *= size
    check(hip, s)


@pytest.mark.parametrize("lens", [(7,), (90,)], ids=["short", "long"])
def test_columns_of_unlike_sizes(hip, lens):
    """A column's error is bounded by its own size, tokens' sizes growing and falling."""
    s = inputs(lens, 1, 1, 128, 48)
    size = 10.0 ** torch.linspace(-9, 9, 48, device=DEV)
    s["v"] *= size
    s["state"] *= size
    check(hip, s)


@pytest.mark.parametrize("lens", [(9,), (80,)], ids=["short", "long"])
def test_without_norm(hip, lens):
    """Keys as given, of length 1 at most; queries of any length."""
    s = inputs(lens, 1, 2, 128, 64)
    s["k"] = s["k"] / s["k"].norm(dim=-1, keepdim=True) * 0.999
    s["q"] *= 37.0
    check(hip, s, norm=False, scale=0.25)


@pytest.mark.parametrize("lens", [(9,), (80,)], ids=["short", "long"])
def test_equal_keys_and_zero_rows(hip, lens):
    s = inputs(lens, 1, 1, 128, 32)
    s["k"][:] = s["k"][0]
    s["k"][3] = 0
    s["q"][5] = 0
    s["v"][6] = 0
    s["beta"][7] = 0
    s["beta"][8] = 1
    check(hip, s)


@pytest.mark.parametrize("most", [1, 16, 70])
def test_limits(hip, most):
    """The first limits[n] tokens only; rows past them are left, and what lies there
    is not looked at."""
    lens = [most, max(1, most // 2), most, most, most]
    limits = [0, lens[1], 1, most, most // 2]
    s = inputs(lens, 2, 2, 128, 64, BF16, extra=5)
    s["v"][-5:] = math.nan
    s["k"][-5:] = math.nan
    s["gate"][-5:] = math.nan
    at = 0
    for n, length in enumerate(lens):
        s["q"][at + limits[n]:at + length] = math.nan
        at += length
    check(hip, s, limits=limits)
    check(hip, s, limits=[x + 1000 if x == lens[n] else x for n, x in enumerate(limits)])


@pytest.mark.parametrize("lens", [(1, 1, 1), (5, 0, 9), (64, 33, 40)],
                         ids=lambda x: "_".join(map(str, x)))
def test_in_place_and_slots(hip, lens):
    """States in place in a pool of more, others untouched; same bits as apart."""
    k3x, ctx = hip
    s = inputs(lens, 1, 2, 128, 128, BF16)
    _, apart = check(hip, s)
    pool = torch.randn((7, 2, 128, 128), device=DEV, generator=gen(4))
    before = pool.clone()
    index = torch.tensor([5, 0, 3], dtype=torch.int32, device=DEV)
    pool[index.long()] = s["state"]
    st, out, _ = call(hip, s, state_in=pool, state_out=pool, slots=7, slot_index=index)
    assert st == 0 and ctx.synchronize() == 0
    assert torch.equal(pool[index.long()], apart)
    rest = [1, 2, 4, 6]
    assert torch.equal(pool[rest], before[rest])


@pytest.mark.parametrize("lens", [(1, 1), (40, 7)], ids=["short", "long"])
def test_without_states(hip, lens):
    """No state before: zeros.  None after: nothing written, one state read by both."""
    k3x, ctx = hip
    s = inputs(lens, 1, 2, 64, 64)
    check(hip, s, state_in=None)
    check(hip, s, state_out=None)
    one = s["state"][:1].clone()
    index = torch.zeros(2, dtype=torch.int32, device=DEV)
    st, out, _ = call(hip, s, state_in=one, state_out=None, slots=1, slot_index=index)
    assert st == 0 and ctx.synchronize() == 0
    s["state"][1] = s["state"][0]
    st, out2, _ = call(hip, s, state_out=None)
    assert st == 0 and ctx.synchronize() == 0
    assert torch.equal(out, out2)


def test_uniform_without_offsets(hip):
    k3x, ctx = hip
    for L in (1, 50):
        s = inputs((L,) * 3, 1, 2, 64, 64)
        st, out, S = call(hip, s)
        st2, out2, S2 = call(hip, s, offsets=None)
        assert st == st2 == 0 and ctx.synchronize() == 0
        assert torch.equal(out, out2) and torch.equal(S, S2)


@pytest.mark.parametrize("lens", [(1, 1), (45, 20)], ids=["short", "long"])
@pytest.mark.parametrize("dtype", [F32, BF16], ids=["fp32", "bf16"])
def test_rows_of_a_projection(hip, lens, dtype):
    """q, k and v as parts of one projection's rows, off 16-byte alignment; out too."""
    k3x, ctx = hip
    Hk, H, K, V = 2, 4, 64, 32
    s = inputs(lens, Hk, H, K, V, dtype)
    st, want, S = call(hip, s)
    T = sum(lens)
    row = torch.randn((T, 3 + 2 * Hk * K + H * V + 5), device=DEV, generator=gen(2)).to(dtype)
    parts = {}
    at = 3
    for x, h, d in (("q", Hk, K), ("k", Hk, K), ("v", H, V)):
        row[:, at:at + h * d] = s[x].reshape(T, -1)
        parts[x] = row[:, at:at + h * d].unflatten(1, (h, d))
        at += h * d
    wide = torch.full((T, H * V + 9), -7.0, device=DEV).to(dtype)
    st2, out, S2 = call(hip, dict(s, **parts), out=wide[:, 1:1 + H * V].unflatten(1, (H, V)))
    assert st == st2 == 0 and ctx.synchronize() == 0
    assert torch.equal(out, want) and torch.equal(S, S2)
    assert (wide[:, 0] == -7).all() and (wide[:, 1 + H * V:] == -7).all()


@pytest.mark.parametrize("longest", [0, 1, 1 << 20])
def test_longest_is_only_a_hint(hip, longest):
    check(hip, inputs((1, 80, 3), 1, 1, 128, 32, BF16), longest=longest)


def test_split_of_a_sequence(hip):
    """A prompt in two chunks, the second from the first's state."""
    k3x, ctx = hip
    whole = inputs((150,), 1, 2, 128, 64, BF16)
    out, S = check(hip, whole)
    for cut in (1, 32, 77, 149):
        a = {x: whole[x][:cut] if whole[x] is not None and x in "qkvbetagate" else whole[x]
             for x in whole}
        b = {x: whole[x][cut:] if whole[x] is not None and x in "qkvbetagate" else whole[x]
             for x in whole}
        a["lens"], b["lens"] = [cut], [150 - cut]
        for part in (a, b):
            part["offsets"] = torch.tensor([0, part["lens"][0]], dtype=torch.int32, device=DEV)
        st, o1, S1 = call(hip, a)
        b["state"] = S1
        st2, o2, S2 = call(hip, b)
        assert st == st2 == 0 and ctx.synchronize() == 0
        want, Sw, tol, stol = definition(whole, 128 ** -0.5)
        close(torch.cat([o1, o2]), want, tol, BF16)
        close(S2, Sw, stol)


@pytest.mark.parametrize("lens", [(2, 2), (40, 40)], ids=["short", "long"])
def test_bad_offsets_and_slots_are_latched(hip, lens):
    """Nothing of the sequences concerned is written."""
    k3x, ctx = hip
    s = inputs(lens, 1, 1, 64, 32)
    T = sum(lens)
    for cu in ([0, T + 1, T], [T, 1, T], [0, 1, T + 7]):
        bad = dict(s, offsets=torch.tensor(cu, dtype=torch.int32, device=DEV))
        st, out, S = call(hip, bad)
        assert st == 0 and ctx.synchronize() == k3x.ERR_INVALID_STATE
    for index in ([0, 2], [-1, 0], [1, 1]):
        st, out, S = call(hip, s, slot_index=torch.tensor(index, dtype=torch.int32, device=DEV))
        assert st == 0 and ctx.synchronize() == k3x.ERR_INVALID_STATE
        if index == [1, 1]:
            assert (S == -7).all() and (out == -7).all()
    check(hip, s)


@pytest.mark.parametrize("lens", [(4,), (70,)], ids=["short", "long"])
@pytest.mark.parametrize("what", ["q", "k", "v", "beta", "gate"])
@pytest.mark.parametrize("value", [math.nan, math.inf])
def test_values_that_are_not_finite_are_latched(hip, lens, what, value):
    k3x, ctx = hip
    s = inputs(lens, 1, 2, 64, 32)
    s[what].view(lens[0], -1)[lens[0] - 2, 3 % s[what][0].numel()] = value
    st, _, _ = call(hip, s)
    assert st == 0 and ctx.synchronize() == k3x.ERR_INVALID_MXFP4
    check(hip, inputs(lens, 1, 2, 64, 32))


@pytest.mark.parametrize("lens", [(1,), (4,), (70,)], ids=["one", "short", "long"])
@pytest.mark.parametrize("value", [math.nan, math.inf])
def test_state_that_is_not_finite_is_latched(hip, lens, value):
    k3x, ctx = hip
    s = inputs(lens, 1, 2, 64, 32)
    s["state"][0, 1, 63, 31] = value
    st, _, _ = call(hip, s)
    assert st == 0 and ctx.synchronize() == k3x.ERR_INVALID_MXFP4
    check(hip, inputs(lens, 1, 2, 64, 32))


def test_growing_gate_is_latched(hip):
    k3x, ctx = hip
    for lens in ((4,), (70,)):
        s = inputs(lens, 1, 1, 64, 32)
        s["gate"][2, 0, 5] = 1e-3
        st, _, _ = call(hip, s)
        assert st == 0 and ctx.synchronize() == k3x.ERR_INVALID_MXFP4


def test_no_tokens(hip):
    """An empty batch: states are copied."""
    k3x, ctx = hip
    s = inputs((0, 0), 1, 1, 32, 16)
    st, _, S = call(hip, s)
    assert st == 0 and ctx.synchronize() == 0
    assert torch.equal(S, s["state"])


@pytest.mark.parametrize("lens", [(1,) * 5, (75, 40)], ids=["short", "long"])
def test_captured(hip, lens):
    """Captured once; replays on changed inputs equal eager calls, bit for bit."""
    k3x, _ = hip
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        ctx = k3x.Context(0)
        own = (k3x, ctx)
        s = inputs(lens, 1, 2, 128, 64, BF16)
        p = k3x.make_delta_params(s["q"], s["k"], s["v"], len(lens), gate=s["gate"], scale=0.1,
                                  norm_epsilon=EPS, longest=max(lens))
        need = k3x.delta_workspace_bytes(p)
        ws = torch.empty((need,), dtype=torch.uint8, device=DEV) if need else None
        out, S = torch.zeros_like(s["v"]), torch.zeros_like(s["state"])
        graph = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, stream=stream):
            assert k3x.delta_rule(ctx, p, s["q"], s["k"], s["v"], s["beta"], out, gate=s["gate"],
                                  offsets=s["offsets"], state_in=s["state"], state_out=S,
                                  workspace=ws) == 0
        for i in range(3):
            s["v"].copy_(torch.randn(s["v"].shape, device=DEV, generator=gen(50 + i)))
            graph.replay()
            got = out.clone(), S.clone()
            st, out2, S2 = call(own, s, scale=0.1)
            assert st == 0 and ctx.synchronize() == 0
            assert torch.equal(got[0], out2) and torch.equal(got[1], S2)
        ctx.close()


def test_two_calls_at_once(hip):
    """Two contexts on two streams, a workspace each."""
    k3x, _ = hip
    s = [inputs((130, 60), 1, 2, 128, 128, BF16, seed=i) for i in range(2)]
    want = [call(hip, x) for x in s]
    assert hip[1].synchronize() == 0
    streams = [torch.cuda.Stream() for _ in s]
    torch.cuda.synchronize()
    ctxs = []
    for stream in streams:
        with torch.cuda.stream(stream):
            ctxs.append(k3x.Context(0))
    for _ in range(4):
        got = []
        for x, ctx, stream in zip(s, ctxs, streams):
            with torch.cuda.stream(stream):
                got.append(call((k3x, ctx), x))
        for ctx in ctxs:
            assert ctx.synchronize() == 0
        for a, b in zip(got, want):
            assert torch.equal(a[1], b[1]) and torch.equal(a[2], b[2])
    for ctx in ctxs:
        ctx.close()


@pytest.mark.parametrize("lens", [(1, 1), (3, 40)], ids=["short", "long"])
def test_states_past_32_bits(hip, lens):
    """2^32 elements and more of states; the last one of them and the first."""
    k3x, ctx = hip
    H, K, V = 32, 128, 128
    slots = 2 ** 32 // (H * K * V) + 2
    s = inputs(lens, 32, H, K, V, BF16)
    index = torch.tensor([slots - 1, 0], dtype=torch.int32, device=DEV)
    states = torch.empty((slots, H, K, V), device=DEV)
    for n, slot in enumerate((slots - 1, 0)):
        states[slot].copy_(s["state"][n])
    st, out, _ = call(hip, s, slot_index=index, state_in=states, state_out=states, slots=slots)
    assert st == 0 and ctx.synchronize() == 0
    want, S, tol, stol = definition(s, K ** -0.5)
    close(out, want, tol, BF16)
    for n, slot in enumerate((slots - 1, 0)):
        close(states[slot], S[n], stol[n])


@pytest.mark.parametrize("lens", [(2, 3), (2, 130)], ids=["short", "long"])
def test_rows_past_32_bits(hip, lens):
    """Rows 2^24 elements apart, the longest stride: the long ones 2^32 bytes from end to end."""
    T, stride = sum(lens), 2 ** 24
    s = inputs(lens, 1, 2, 64, 64, BF16)
    wide = torch.empty((T, stride), dtype=BF16, device=DEV)
    at = 0
    for x, n in (("q", 64), ("k", 64), ("v", 128)):
        rows = wide[:, at:at + n].unflatten(1, (-1, 64))
        rows.copy_(s[x])
        s[x] = rows
        at += n
    out = wide[:, stride - 128:].unflatten(1, (2, 64))
    k3x, ctx = hip
    st, out, S = call(hip, s, out=out)
    assert st == 0 and ctx.synchronize() == 0
    want, Sw, tol, stol = definition(s, 64 ** -0.5)
    close(out, want, tol, BF16)
    close(S, Sw, stol)


def quiet(s, tokens):
    """The first `tokens` rows without values, under a decay that empties no state."""
    s["v"][:tokens] = 0
    if s["gate"] is not None:
        s["gate"][:] = -0.7
    return s


@pytest.mark.parametrize("longest", [1, 1 << 20], ids=["tokens", "chunks"])
@pytest.mark.parametrize("gate", ["head", "channel"])
@pytest.mark.parametrize("tokens,decay", [(96, -1.6), (192, -0.7), (1000, -0.7)])
def test_values_after_a_long_decay(hip, tokens, decay, gate, longest):
    """Nothing is written for a while, so that the state all but vanishes; then values of
    size one."""
    s = quiet(inputs((tokens + 70,), 1, 2, 128, 48, BF16, gate), tokens)
    s["gate"][:] = decay
    check(hip, s, longest=longest)


@pytest.mark.parametrize("longest", [1, 1 << 20], ids=["tokens", "chunks"])
@pytest.mark.parametrize("gate", ["none", "head", "channel"])
@pytest.mark.parametrize("size", [1e-30, 1e-36, 1e-40, 1e30, 1e36])
def test_state_and_values_of_unlike_sizes(hip, size, gate, longest):
    """A state next to nothing, or far above the values that follow; every other column as
    large as they are."""
    s = inputs((50,), 1, 2, 64, 48, gate=gate)
    s["state"][..., ::2] *= size
    check(hip, s, longest=longest)


@pytest.mark.parametrize("longest", [1, 1 << 20], ids=["tokens", "chunks"])
@pytest.mark.parametrize("dtype", [F32, BF16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("gate", ["none", "head", "channel"])
def test_values_near_the_largest(hip, gate, dtype, longest):
    s = quiet(inputs((90,), 1, 2, 128, 48, dtype, gate), 90)
    for t in (5, 40):
        s["v"][t] = (1.5e37 * (2 * torch.rand(s["v"][t].shape, device=DEV, generator=gen(t)) - 1)
                     ).to(dtype)
    s["state"][:] = 0
    check(hip, s, longest=longest)


@pytest.mark.parametrize("gate", ["head", "channel"])
def test_long_decay_over_two_calls(hip, gate):
    """The second call starts from the state that is left, around the smallest numbers."""
    k3x, ctx = hip
    whole = quiet(inputs((250,), 1, 2, 128, 48, BF16, gate), 130)
    a = {x: whole[x][:130] if x in ("q", "k", "v", "beta", "gate") else whole[x] for x in whole}
    b = {x: whole[x][130:] if x in ("q", "k", "v", "beta", "gate") else whole[x] for x in whole}
    a["lens"], b["lens"] = [130], [120]
    for part in (a, b):
        part["offsets"] = torch.tensor([0, part["lens"][0]], dtype=torch.int32, device=DEV)
    _, b["state"] = check(hip, a)
    check(hip, b)


@pytest.mark.parametrize("in_place", [False, True], ids=["apart", "in_place"])
def test_sequences_of_no_tokens_keep_their_states(hip, in_place):
    """A state is copied bit for bit, whatever its columns span, also beside long sequences
    and where a limit leaves no token."""
    k3x, ctx = hip
    s = inputs((0, 80, 3, 40), 1, 2, 128, 48)
    s["state"] *= 10.0 ** torch.linspace(-42, 36, 128, device=DEV)[:, None]
    s["state"][0, 1, 3, 7], s["state"][0, 1, 4, 7] = math.nan, -math.inf
    before = s["state"].clone()
    st, _, S = call(hip, s, limits=[5, 0, 0, 7], **(dict(state_out=s["state"]) if in_place else {}))
    assert st == 0 and ctx.synchronize() == 0
    assert torch.equal(S[:3].view(torch.int32), before[:3].view(torch.int32))
    assert not torch.equal(S[3], before[3])


FAULTS = ["q", "v", "state", "slot", "twice"]


@pytest.mark.parametrize("fault", FAULTS)
@pytest.mark.parametrize("length,N", [(1, 700), (40, 100)], ids=["short", "long"])
@pytest.mark.parametrize("gate", ["head", "channel"])
def test_a_fault_leaves_the_other_sequences_whole(hip, gate, length, N, fault):
    """States in place: sequences beside an unfit one are those of a call without it, all
    their heads and columns, more of them than run at once.  What is enqueued after the
    call does nothing until the error is read."""
    k3x, ctx = hip
    s = inputs((length,) * N, 1, 8, 128, 128, BF16, gate)
    pool = torch.empty((N + 3, 8, 128, 128), device=DEV)
    pool[:N].copy_(s["state"])
    pool[N:] = -7.0
    clean, index = pool.clone(), torch.arange(N, dtype=torch.int32, device=DEV)
    st, want, _ = call(hip, s, state_in=clean, state_out=clean, slots=N + 3, slot_index=index)
    assert st == 0 and ctx.synchronize() == 0
    fit, code = torch.ones(N, dtype=torch.bool, device=DEV), k3x.ERR_INVALID_MXFP4
    fit[0] = False
    if fault == "state":
        pool[0, 3, 5] = math.inf
    elif fault in ("slot", "twice"):
        index[0] = N + 3 if fault == "slot" else N - 1
        fit[N - 1] = fault == "slot"
        code = k3x.ERR_INVALID_STATE
    else:
        s[fault][length // 2, 0, 2] = math.nan
    before = pool.clone()
    st, out, _ = call(hip, s, state_in=pool, state_out=pool, slots=N + 3, slot_index=index)
    assert st == 0
    later = torch.full((2, 4), -7, dtype=torch.int32, device=DEV)
    weights = torch.full((2, 4), -7.0, device=DEV)
    assert k3x.route(ctx, k3x.make_route_params(2, 64, 4), torch.zeros((2, 64), device=DEV), later,
                     weights) == 0
    st, out2, S2 = call(hip, dict(s, lens=[length], offsets=s["offsets"][:2], state=clean[:1]))
    assert st == 0
    assert ctx.synchronize() == code
    assert (later == -7).all() and (weights == -7).all()
    assert (out2 == -7).all() and (S2 == -7).all()
    assert torch.equal(pool[:N][fit], clean[:N][fit])
    assert torch.equal(out.unflatten(0, (N, length))[fit], want.unflatten(0, (N, length))[fit])
    assert (pool[N:] == -7).all()
    if code == k3x.ERR_INVALID_STATE:  # nothing of the unfit ones is written
        assert torch.equal(pool[:N][~fit], before[:N][~fit])
        assert (out.unflatten(0, (N, length))[~fit] == -7).all()
    assert ctx.synchronize() == 0


@pytest.mark.parametrize("cu", [[0, 41, 40, 120], [120, 40, 80, 120], [0, 40, 80, 79],
                                [1 << 31, 0, 60, 120]], ids=["middle", "first", "last", "far"])
@pytest.mark.parametrize("gate", ["head", "channel"])
def test_falling_offsets_in_chunks(hip, gate, cu):
    """No sequence of the call is touched: the workspace holds what an earlier call left."""
    k3x, ctx = hip
    s = inputs((40, 40, 40), 1, 2, 64, 32, BF16, gate)
    pool = s["state"].clone()
    cu = [x - (1 << 32) if x >> 31 else x for x in cu]
    st, out, _ = call(hip, s, state_in=pool, state_out=pool,
                      offsets=torch.tensor(cu, dtype=torch.int32, device=DEV))
    assert st == 0 and ctx.synchronize() == k3x.ERR_INVALID_STATE
    assert torch.equal(pool, s["state"]) and (out == -7).all()
    check(hip, s)


@pytest.mark.parametrize("what", ["q", "k"])
@pytest.mark.parametrize("gate", ["head", "channel"])
@pytest.mark.parametrize("longest", [1, 1 << 20], ids=["tokens", "chunks"])
def test_norms_past_the_range_are_latched(hip, longest, gate, what):
    """A row whose sum of squares is no fp32 number is not taken for one of length 0."""
    k3x, ctx = hip
    s = inputs((40,), 1, 2, 64, 32, BF16, gate)
    s[what][20] = (s[what][20].float() * 1e20).to(BF16)
    st, _, _ = call(hip, s, longest=longest)
    assert st == 0 and ctx.synchronize() == k3x.ERR_INVALID_MXFP4
    s[what][20] = (s[what][20].float() * 1e-3).to(BF16)
    check(hip, s, longest=longest)


@pytest.mark.parametrize("gate", ["head", "channel"])
@pytest.mark.parametrize("size", [1e-20, 1e20, 1e34])
@pytest.mark.parametrize("longest", [1, 1 << 20], ids=["tokens", "chunks"])
def test_queries_of_any_size_without_norm(hip, longest, size, gate):
    s = inputs((45,), 1, 2, 64, 32, gate=gate)
    s["k"] = s["k"] / s["k"].norm(dim=-1, keepdim=True) * 0.999
    s["q"] *= size
    check(hip, s, norm=False, scale=0.5, longest=longest)


def owned_rows(lens, sequences):
    at, rows = 0, []
    for n, length in enumerate(lens):
        if n in sequences:
            rows += range(at, at + length)
        at += length
    return rows


@pytest.mark.parametrize("in_place", [False, True], ids=["apart", "in_place"])
@pytest.mark.parametrize("lens", [(2, 2), (40, 40)], ids=["short", "long"])
@pytest.mark.parametrize("index,unfit", [([0, 4], [1]), ([-1, 2], [0]), ([3, 3], [0, 1]),
                                         ([1 << 30, 4], [0, 1])])
def test_slots_that_are_no_states(hip, index, unfit, lens, in_place):
    """Rows of a sequence without a state and states without a sequence stay as they were,
    beyond the last one of the call too."""
    k3x, ctx = hip
    s = inputs(lens, 1, 1, 64, 32)
    room = torch.full((9, 1, 64, 32), -7.0, device=DEV)
    pool = room[1:5]
    fresh = torch.full_like(room, -7.0)
    pool[:2].copy_(s["state"])
    before = room.clone()
    st, out, _ = call(hip, s, state_in=pool, state_out=pool if in_place else fresh[1:5], slots=4,
                      slot_index=torch.tensor(index, dtype=torch.int32, device=DEV))
    assert st == 0 and ctx.synchronize() == k3x.ERR_INVALID_STATE
    assert (out[owned_rows(lens, unfit)] == -7).all()
    mine = [1 + x for n, x in enumerate(index) if n not in unfit]
    rest = [x for x in range(9) if x not in mine]
    assert torch.equal(room[rest], before[rest])
    assert (fresh[rest] == -7).all()


@pytest.mark.parametrize("lens", [(2, 2), (40, 40)], ids=["short", "long"])
def test_offsets_past_the_rows(hip, lens):
    """Sequences that end behind the last row read and write nothing, nor do those that
    fall; what lies around the rows and the states stays as it was."""
    k3x, ctx = hip
    s = inputs(lens, 1, 1, 64, 32, extra=50)
    T = sum(lens)
    room = dict(out=torch.full((T + 50, 1, 32), -7.0, device=DEV),
                state=torch.full((6, 1, 64, 32), -7.0, device=DEV))
    few = {x: y[:T] if x in ("q", "k", "v", "beta", "gate") else y for x, y in s.items()}
    for cu, unfit in (([0, T // 2, T + 7], [1]), ([T + 1, T + 2, T + 3], [0, 1]),
                      ([0, T + 1, T], [0, 1]), ([-9, 0, T // 2], [0])):
        for x in room.values():
            x[:] = -7.0
        st, _, _ = call(hip, few, out=room["out"][:T], state_out=room["state"][:2],
                        offsets=torch.tensor(cu, dtype=torch.int32, device=DEV))
        assert st == 0 and ctx.synchronize() == k3x.ERR_INVALID_STATE
        assert (room["out"][T:] == -7).all() and (room["state"][2:] == -7).all()
        assert (room["state"][unfit] == -7).all()
        if cu[0] == 0 and cu[1] <= cu[2]:
            assert (room["out"][T // 2:T] == -7).all()


@pytest.mark.parametrize("gate", ["none", "head", "channel"])
@pytest.mark.parametrize("norm", [True, False], ids=["norm", "given"])
def test_values_that_grow_within_a_chunk(hip, gate, norm):
    """Tokens before larger ones of their chunk, up to 2^13 times as large: within the bound
    that their own and earlier sizes give."""
    s = inputs((96,), 1, 2, 64, 48, gate=gate)
    if not norm:
        s["k"] = s["k"] / s["k"].norm(dim=-1, keepdim=True) * 0.999
    s["state"][:] = 0
    s["v"] = s["v"].sign() * (1 + s["v"].abs().clamp(max=1))
    s["v"] *= (2.0 ** (torch.arange(96, device=DEV) % 32 * 0.4))[:, None, None]
    check(hip, s, norm=norm)


@pytest.mark.parametrize("lens", [(1,) * 5, (75, 40, 33)], ids=["short", "long"])
def test_captured_in_place(hip, lens):
    """Replays move the states on; one that meets an unfit sequence moves the others', the
    next does nothing until the error is read, and those after it run again."""
    k3x, _ = hip
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        ctx = k3x.Context(0)
        s = inputs(lens, 1, 2, 128, 64, BF16)
        p = k3x.make_delta_params(s["q"], s["k"], s["v"], len(lens), gate=s["gate"], scale=0.1,
                                  norm_epsilon=EPS, longest=max(lens))
        need = k3x.delta_workspace_bytes(p)
        ws = torch.empty((need,), dtype=torch.uint8, device=DEV) if need else None
        one, two = s["state"].clone(), s["state"].clone()
        out, out2 = torch.zeros_like(s["v"]), torch.zeros_like(s["v"])

        def run(state, out):
            return k3x.delta_rule(ctx, p, s["q"], s["k"], s["v"], s["beta"], out, gate=s["gate"],
                                  offsets=s["offsets"], state_in=state, state_out=state,
                                  workspace=ws)

        graph = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, stream=stream):
            assert run(one, out) == 0
        for i in range(5):
            s["v"].copy_(torch.randn(s["v"].shape, device=DEV, generator=gen(60 + i)))
            kept = s["v"][0].clone()
            assert run(two, out2) == 0 and ctx.synchronize() == 0
            if i == 2:
                s["v"][0, 0, 0] = math.nan
            graph.replay()
            if i != 2:
                assert ctx.synchronize() == 0
                assert torch.equal(one, two) and torch.equal(out, out2)
                continue
            s["v"][0].copy_(kept)
            after = one.clone()
            graph.replay()
            assert ctx.synchronize() == k3x.ERR_INVALID_MXFP4
            assert torch.equal(one[1:], two[1:]) and torch.equal(one[1:], after[1:])
            assert torch.equal(out[lens[0]:], out2[lens[0]:])
            one[0].copy_(two[0])
            out.copy_(out2)
        del graph
        ctx.close()
