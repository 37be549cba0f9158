"""Routing, the gated delta rule and draft verification together, as a serving
step with drafted tokens uses them: the delta rule over a window of the last
token and the drafts without writing its states, routing and the experts on its
outputs, verification of the drafts against the rows that follow, and the delta
rule again, states written, up to the last accepted token.

Each stage is checked against 64 bits on the stage's own inputs: the delta rule
with the bounds of test_gpu_delta, routes with those of test_gpu_route, tokens
exactly.  The experts' mix is within the experts' bound (test_gpu_few_pairs)
carried through the K weights, the roundings to bf16 of an expert's output and
of the mix (2^-8 each) and the mix's fp32 sum ((K + 1) 2^-24)."""
from __future__ import annotations

import pytest

import test_gpu_delta as delta
import test_gpu_route as routing
import test_gpu_verify as verify

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")
DEV = "cuda:0"
BF16 = torch.bfloat16

HIDDEN, INTER, EXPERTS, TOP_K, VOCAB = 512, 256, 24, 3, 1003
HK, H, K, V = 2, 4, 64, 64


@pytest.fixture(scope="module")
def hip():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    import k3x_amd
    ctx = k3x_amd.Context(0)
    yield k3x_amd, ctx
    ctx.close()


class Step:
    """One layer and an output head, and N users' windows of D drafts."""

    def __init__(self, k3x, ctx, N, D, gate, seed):
        self.k3x, self.ctx, self.N, self.D = k3x, ctx, N, D
        g = delta.gen(seed)

        def n(*shape):
            return torch.randn(shape, device=DEV, generator=g)

        self.s = delta.inputs((D + 1,) * N, HK, H, K, V, BF16, gate, seed=seed)
        self.bank = k3x.Bank(ctx, k3x.LayerShape(HIDDEN, INTER, EXPERTS, 0))
        self.bank.fill_synthetic(seed, 119, 123)
        self.wo = n(H * V, HIDDEN) * 0.5
        self.wr, self.bias = n(HIDDEN, EXPERTS) * 0.1, n(EXPERTS) * 0.05
        self.wv = n(HIDDEN, VOCAB) * 0.1
        T = N * (D + 1)
        self.out, self.again = (torch.full((T, H, V), -7.0, device=DEV).to(BF16) for _ in "ab")
        self.ids = torch.full((T, TOP_K), -7, dtype=torch.int32, device=DEV)
        self.weights = torch.full((T, TOP_K), -7.0, device=DEV)
        self.mix = torch.empty((T, HIDDEN), dtype=BF16, device=DEV)
        self.x = torch.empty_like(self.mix)
        self.logits = torch.empty((T, EXPERTS), device=DEV)
        self.accepted = torch.full((N,), -7, dtype=torch.int32, device=DEV)
        self.limits = torch.full((N,), -7, dtype=torch.int32, device=DEV)
        self.tokens = torch.full((N, D + 1), -7, dtype=torch.int32, device=DEV)
        self.state = self.s["state"].clone()
        self.window = k3x.make_delta_params(self.s["q"], self.s["k"], self.s["v"], N,
                                            gate=self.s["gate"], scale=K ** -0.5,
                                            norm_epsilon=delta.EPS, longest=D + 1)
        need = k3x.delta_workspace_bytes(self.window)
        self.delta_ws = torch.empty((need,), dtype=torch.uint8, device=DEV) if need else None
        self.route = k3x.make_route_params(T, EXPERTS, TOP_K, routed_scale=1.5)
        self.v = dict(target=torch.zeros((N, D + 1, VOCAB), device=DEV))
        self.verify = k3x.make_verify_params(self.v["target"], temperature=0.9)
        need = k3x.verify_workspace_bytes(self.verify)
        self.verify_ws = torch.empty((need,), dtype=torch.uint8, device=DEV)

    def rule(self, out, limits=None, commit=False):
        s = self.s
        self.k3x.check(self.k3x.delta_rule(
            self.ctx, self.window, s["q"], s["k"], s["v"], s["beta"], out, gate=s["gate"],
            offsets=s["offsets"], limits=limits, state_in=self.state,
            state_out=self.state if commit else None, workspace=self.delta_ws), "delta_rule")

    def experts(self):
        k3x = self.k3x
        k3x.check(k3x.route(self.ctx, self.route, self.logits, self.ids, self.weights,
                            bias=self.bias), "route")
        params = k3x.make_params(len(self.ids), TOP_K, 1.0)
        k3x.check(k3x.moe_forward_routed(self.ctx, self.bank, params, self.x, self.ids,
                                         self.weights, self.mix), "experts")

    def verified(self):
        v = self.v
        self.k3x.check(self.k3x.verify_draft(
            self.ctx, self.verify, v["target"], v["tokens"], self.accepted, self.tokens,
            draft=v["draft"], accept_u=v["accept_u"], sample_u=v["sample_u"],
            workspace=self.verify_ws), "verify_draft")
        torch.add(self.accepted, 1, out=self.limits)

    def drafts(self, seed):
        """Drafts that the target accepts now and then."""
        g = delta.gen(seed)
        v, t = self.v, self.v["target"][:, :self.D]
        v["draft"] = t + torch.randn(t.shape, device=DEV, generator=g) * 0.5
        v["tokens"] = torch.distributions.Categorical(logits=v["draft"] / 0.9).sample().to(
            torch.int32)
        v["accept_u"] = torch.rand((self.N, self.D), device=DEV, generator=g)
        v["sample_u"] = torch.rand((self.N,), device=DEV, generator=g)


def check_experts(step):
    x, want = step.x.double(), torch.zeros((len(step.x), HIDDEN), device=DEV).double()
    tol = torch.zeros_like(want)
    for e in range(EXPERTS):
        tok, slot = (step.ids == e).nonzero(as_tuple=True)
        if not len(tok):
            continue
        gate, up, down = (step.bank.dequant_rows(e, m, 0, INTER if m < 2 else HIDDEN).double()
                          for m in range(3))
        gv, uv = x[tok] @ gate.t(), x[tok] @ up.t()
        eps = HIDDEN * 2.0 ** -24
        dg, du = (eps * (x[tok].abs() @ m.abs().t()) for m in (gate, up))
        silu = gv / (1 + torch.exp(-gv))
        act = silu * uv
        dact = 1.1 * (uv.abs() * dg + silu.abs() * du + dg * du) + 2.0 ** -8 * act.abs()
        y = act @ down.t()
        dy = dact @ down.abs().t() + INTER * 2.0 ** -24 * ((act.abs() + dact) @ down.abs().t())
        w = step.weights[tok, slot].double()[:, None]
        want[tok] += w * y
        tol[tok] += w * (dy + (2.0 ** -8 + (TOP_K + 1) * 2.0 ** -24) * (y.abs() + dy))
    err = (step.mix.double() - want).abs()
    assert (err <= tol + 2.0 ** -8 * (want.abs() + tol) + 1e-30).all()


@pytest.mark.parametrize("gate", ["head", "channel"])
@pytest.mark.parametrize("N,D", [(1, 1), (5, 4), (3, 30)])
def test_step(hip, N, D, gate):
    k3x, ctx = hip
    print(f"[gpu-test] speculative step N={N} D={D} {gate}", flush=True)
    step = Step(k3x, ctx, N, D, gate, 7 * N + D)
    before = step.state.clone()
    step.rule(step.out)
    step.x.copy_(step.out.float().flatten(1) @ step.wo)
    step.logits.copy_(step.x.float() @ step.wr)
    step.experts()
    step.v["target"].copy_((step.mix.float() @ step.wv).unflatten(0, (N, D + 1)))
    step.drafts(N + D)
    step.verified()
    assert torch.equal(step.state, before)  # the window has written no state
    step.rule(step.again, limits=step.limits, commit=True)
    assert ctx.synchronize() == 0

    want, _, tol, _ = delta.definition(step.s, K ** -0.5)
    delta.close(step.out, want, tol, BF16)
    ids, weights = routing.plain(step.logits, step.bias, TOP_K, scale=1.5)
    assert torch.equal(step.ids.cpu().long(), ids)
    err = (step.weights.cpu().double() - weights).abs()
    assert (err <= (4 + TOP_K) * 2.0 ** -24 * weights).all()
    check_experts(step)
    accepted, tokens = verify.definition(step.v, False, False, 0.9)
    assert torch.equal(step.accepted.cpu(), accepted)
    assert torch.equal(step.tokens.cpu(), tokens)
    limits = [int(a) + 1 for a in accepted]
    _, state, _, stol = delta.definition(step.s, K ** -0.5, limits=limits)
    delta.close(step.state, state, stol)
    for n in range(N):  # the rows run twice are the window's, the others untouched
        at = n * (D + 1)
        assert torch.equal(step.again[at:at + limits[n]], step.out[at:at + limits[n]])
        assert (step.again[at + limits[n]:at + D + 1] == -7).all()
    step.bank.close()


@pytest.mark.parametrize("D", [3, 30])
def test_captured_step(hip, D):
    """The operators of a step in one graph; replays on changed inputs, from
    the states of the replay before, equal eager steps bit for bit."""
    k3x, _ = hip
    N = 4
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        ctx = k3x.Context(0)
        one, two = (Step(k3x, ctx, N, D, "channel", 3) for _ in range(2))

        def run(step):
            step.rule(step.out)
            step.experts()
            step.verified()
            step.rule(step.again, limits=step.limits, commit=True)

        def fill(step, seed):
            g = delta.gen(seed)
            step.s["v"].copy_(torch.randn(step.s["v"].shape, device=DEV, generator=g))
            step.x.copy_(torch.randn(step.x.shape, device=DEV, generator=g))
            step.logits.copy_(torch.randn(step.logits.shape, device=DEV, generator=g))
            step.v["target"].copy_(torch.randn(step.v["target"].shape, device=DEV, generator=g))

        for step in (one, two):
            fill(step, 1)
        one.drafts(2)
        two.v = {x: y.clone() for x, y in one.v.items()}
        run(two)
        two.state.copy_(one.state)
        two.again.copy_(one.again)  # rows past the accepted ones stay as they were
        assert ctx.synchronize() == 0
        graph = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, stream=stream):
            run(one)
        for i in range(3):
            for step in (one, two):
                fill(step, 10 + i)
            graph.replay()
            run(two)
            assert ctx.synchronize() == 0
            for x in ("out", "ids", "weights", "mix", "accepted", "tokens", "again", "state"):
                assert torch.equal(getattr(one, x), getattr(two, x)), (i, x)
        del graph
        one.bank.close()
        two.bank.close()
        ctx.close()


@pytest.mark.parametrize("gate", ["head", "channel"])
@pytest.mark.parametrize("D", [3, 30])
def test_sequences_left_out_keep_their_states(hip, D, gate):
    """draft_counts leaves sequences out and gives others fewer drafts: the limits made of
    both outputs commit nothing of the former."""
    k3x, ctx = hip
    N = 5
    counts = [D, -1, 0, D - 1, -1]
    step = Step(k3x, ctx, N, D, gate, 11)
    before = step.state.clone()
    g = delta.gen(4)
    step.v["target"].copy_(torch.randn(step.v["target"].shape, device=DEV, generator=g))
    step.drafts(5)
    v = step.v
    assert k3x.verify_draft(
        ctx, step.verify, v["target"], v["tokens"], step.accepted, step.tokens, draft=v["draft"],
        draft_counts=torch.tensor(counts, dtype=torch.int32, device=DEV),
        accept_u=v["accept_u"], sample_u=v["sample_u"], workspace=step.verify_ws) == 0
    step.limits = torch.where(step.tokens[:, 0] == -1, 0, step.accepted + 1)
    assert step.limits.dtype == torch.int32
    step.rule(step.again, limits=step.limits, commit=True)
    assert ctx.synchronize() == 0
    accepted, tokens = verify.definition(v, False, False, 0.9, counts)
    assert torch.equal(step.accepted.cpu(), accepted) and torch.equal(step.tokens.cpu(), tokens)
    limits = [0 if c == -1 else int(a) + 1 for c, a in zip(counts, accepted)]
    assert step.limits.tolist() == limits
    out, state, tol, stol = delta.definition(step.s, K ** -0.5, limits=limits)
    delta.close(step.state, state, stol)
    for n in range(N):
        at = n * (D + 1)
        rows = slice(at, at + limits[n])
        delta.close(step.again[rows], out[rows], tol[rows], BF16)
        assert (step.again[at + limits[n]:at + D + 1] == -7).all()
        if counts[n] == -1:
            assert torch.equal(step.state[n], before[n])
        else:
            assert not torch.equal(step.state[n], before[n])
    step.bank.close()
