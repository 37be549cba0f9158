"""Latent attention, its cache and the adjustment of logits together, as a serving step with
drafted tokens uses them: a prompt chunk is stored, the prefix before it read back and expanded,
and attended to; then windows of the last token and the drafts are stored and attend to the
cache, and their logits are adjusted and verified.

Each stage is checked against 64 bits on the stage's own inputs, with the bounds of test_gpu_mla,
test_gpu_mla_prompt, test_gpu_logits and test_gpu_verify."""
from __future__ import annotations

import pytest

import mla_reference as ref
import test_gpu_logits as adjusted
import test_gpu_mla as mla
import test_gpu_verify as verify

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")
DEV = "cuda:0"
BF16 = torch.bfloat16
L, R, HIDDEN, DN, DV, VOCAB, EPS = 128, 32, 256, 64, 64, 1003, 1e-6
F32_EPS = float(torch.tensor(EPS))


@pytest.fixture(scope="module")
def hip():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    import k3x_amd
    ctx = k3x_amd.Context(0)
    yield k3x_amd, ctx
    ctx.close()


def written(latent, gamma, fmt):
    """The values that a stored latent stands for."""
    x = latent.cpu().double()
    x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + F32_EPS) * gamma.cpu().double()
    return ref.encode(x.float().to(latent.dtype), torch.zeros((len(x), 0)), fmt)[1]


class Layer:
    """A layer's weights, a cache of `lens` tokens a sequence with room for `more`, and windows of
    D drafts."""

    def __init__(self, k3x, ctx, lens, H, D, fmt, seed, more=64, page=16):
        self.k3x, self.ctx, self.H, self.D, self.fmt = k3x, ctx, H, D, fmt
        N = self.N = len(lens)
        self.lens = lens
        g = verify.gen(seed)

        def n(*shape, by=1.0):
            return torch.randn(shape, device=DEV, generator=g) * by

        self.gamma = 1 + 0.2 * n(L)
        self.wq = n(HIDDEN, H * (DN + R), by=0.06)
        self.wc = n(HIDDEN, L + R, by=0.06)
        self.wk, self.wv = n(H, DN, L, by=0.1), n(H, DV, L, by=0.1)
        self.wo = n(H * DV, VOCAB, by=0.2)
        width = -(-(max(lens) + more) // page)
        cache = ref.make_cache([width * page] * N, L, R, page, fmt, seed=seed)
        for i in range(N):  # what is past the lengths is of no use to any call
            cache["rows"][i] = tuple(r[:lens[i]] for r in cache["rows"][i])
        self.rows = cache["rows"]
        self.cache = mla.to_device(cache)
        self.at = mla.ints(lens)
        self.scale = float(torch.tensor((DN + R) ** -0.5))
        T = self.T = N * (D + 1)
        self.new = n(T, L + R).to(BF16)
        self.q = n(T, H, L + R).to(BF16)
        self.out = torch.full((T, H, L), -7.0, dtype=BF16, device=DEV)
        self.back = torch.full((T, L), -7.0, dtype=BF16, device=DEV)
        self.lse = torch.full((T, H), -7.0, device=DEV)
        self.p = mla.params(k3x, self.cache, T, H, self.scale, EPS, D + 1)
        need = k3x.mla_attention_workspace_bytes(self.p)
        self.ws = torch.empty((need,), dtype=torch.uint8, device=DEV)
        self.logits = n(N, D + 1, VOCAB)
        s = adjusted.make(N, D, VOCAB, seed=seed)
        s.pop("logits")
        words = torch.rand((3, 32 * -(-VOCAB // 32)), generator=ref.gen(seed)) < 0.8
        s["masks"] = (words.view(3, -1, 32) * (1 << torch.arange(32))).sum(-1).to(torch.int32)
        self.s = {k: tuple(t.to(DEV) for t in v) if isinstance(v, tuple) else v.to(DEV)
                  for k, v in s.items()}
        self.adjusted = torch.zeros_like(self.logits)
        self.verify = k3x.make_verify_params(self.logits, temperature=0.9)
        self.draft = n(N, D, VOCAB)
        self.uniforms = (torch.rand((N, D), device=DEV, generator=g),
                         torch.rand((N,), device=DEV, generator=g))
        self.accepted = torch.full((N,), -7, dtype=torch.int32, device=DEV)
        self.tokens = torch.full((N, D + 1), -7, dtype=torch.int32, device=DEV)
        need = k3x.verify_workspace_bytes(self.verify)
        self.verify_ws = torch.empty((need,), dtype=torch.uint8, device=DEV)

    def store(self):
        c = self.cache
        self.k3x.check(self.k3x.mla_store(
            self.ctx, self.p, self.new[:, :L], c["pool"], c["table"], self.at,
            rotary=self.new[:, L:], gamma=self.gamma), "mla_store")

    def attend(self):
        c = self.cache
        self.k3x.check(self.k3x.mla_attention(
            self.ctx, self.p, self.q, c["pool"], c["table"], self.at, self.out, lse=self.lse,
            workspace=self.ws), "mla_attention")

    def load(self):
        c = self.cache
        self.k3x.check(self.k3x.mla_load(self.ctx, self.p, c["pool"], c["table"], self.at,
                                         self.back), "mla_load")

    def adjust(self):
        self.k3x.check(self.k3x.adjust_logits(
            self.ctx, self.k3x.make_logits_params(self.logits), self.logits, self.adjusted,
            **self.s), "adjust_logits")

    def verified(self):
        self.k3x.check(self.k3x.verify_draft(
            self.ctx, self.verify, self.adjusted, self.s["drafts"], self.accepted, self.tokens,
            draft=self.draft, accept_u=self.uniforms[0], sample_u=self.uniforms[1],
            workspace=self.verify_ws), "verify_draft")

    def step(self):
        """The window's calls, on what the buffers hold."""
        self.store()
        self.load()
        self.attend()
        self.adjust()
        self.verified()


@pytest.mark.parametrize("fmt", ["16bit", "mxfp8", "mxfp4"])
@pytest.mark.parametrize("H,lens,D", [(4, [0, 37, 100], 3), (16, [250], 1)], ids=str)
def test_prompt_and_window(hip, fmt, H, lens, D):
    k3x, ctx = hip
    print(f"[gpu-test] prompt and window H={H} {lens} D={D} {fmt}", flush=True)
    y = Layer(k3x, ctx, lens, H, D, fmt, 5 + H)
    c, N = y.cache, y.N

    # A chunk of the prompt: its rows stored, the prefix and they read back, expanded, attended to.
    chunk = [21, 1, 40][:N]
    total = [a + b for a, b in zip(lens, chunk)]
    T, S = sum(chunk), sum(total)
    x = torch.randn((T, HIDDEN), generator=ref.gen(1)).to(DEV)
    new = (x @ y.wc).to(BF16)
    p = mla.params(k3x, c, T, eps=EPS)
    k3x.check(k3x.mla_store(ctx, p, new[:, :L], c["pool"], c["table"], mla.ints(total),
                            rotary=new[:, L:], offsets=mla.offsets_of(chunk), gamma=y.gamma),
              "mla_store")
    latent = torch.empty((S, L), dtype=BF16, device=DEV)
    rotary = torch.empty((S, R), dtype=BF16, device=DEV)
    k3x.check(k3x.mla_load(ctx, mla.params(k3x, c, S), c["pool"], c["table"], mla.ints(total),
                           latent, rotary=rotary, offsets=mla.offsets_of(total)), "mla_load")
    q = (x @ y.wq).view(T, H, DN + R).to(BF16)
    kv = torch.cat([(latent.float() @ w.flatten(0, 1).t()).view(S, H, -1).to(BF16)
                    for w in (y.wk, y.wv)], 2)
    out = torch.empty((T, H, DV), dtype=BF16, device=DEV)
    pp = k3x.make_mla_prompt_params(q, kv[..., :DN], kv[..., DN:], N, rotary=rotary,
                                    scale=y.scale)
    k3x.check(k3x.mla_prompt(ctx, pp, q, kv[..., :DN], kv[..., DN:], out, rotary=rotary,
                             offsets=mla.offsets_of(chunk), key_offsets=mla.offsets_of(total)),
              "mla_prompt")
    assert ctx.synchronize() == 0
    values = written(new[:, :L], y.gamma, fmt)
    at = 0
    for n in range(N):
        y.rows[n] = tuple(torch.cat([a, b[at:at + chunk[n]]]) for a, b in
                          zip(y.rows[n], (values, new[:, L:].cpu().double())))
        at += chunk[n]
    assert torch.equal(latent.cpu().double(), torch.cat([r[0] for r in y.rows]))
    assert torch.equal(rotary.cpu().double(), torch.cat([r[1] for r in y.rows]))
    want, _, tol, _ = ref.prompt(q, kv[..., :DN], kv[..., DN:], rotary, chunk, total, True,
                                 y.scale)
    assert ref.close(out, want, tol) <= 1

    # The window: its rows are the sequences' last D + 1.
    lens = [n + D + 1 for n in total]
    y.at.copy_(mla.ints(lens))
    q = torch.randn((y.T, H, DN), generator=ref.gen(2)).to(DEV)
    y.q[..., :L] = torch.einsum("thd,hdl->thl", q, y.wk).to(BF16)
    y.store()
    y.attend()
    y.load()
    o = torch.einsum("thl,hdl->thd", y.out.float(), y.wv).flatten(1)
    y.logits.copy_((o @ y.wo).view(N, D + 1, VOCAB))
    y.draft.copy_(y.logits[:, :D] + 0.5 * y.draft)
    y.s["drafts"].copy_(torch.distributions.Categorical(logits=y.draft / 0.9).sample().int())
    y.adjust()
    y.verified()
    assert ctx.synchronize() == 0
    values = written(y.new[:, :L], y.gamma, fmt)
    assert torch.equal(y.back.cpu().double(), values)
    for n in range(N):
        rows = slice(n * (D + 1), (n + 1) * (D + 1))
        y.rows[n] = tuple(torch.cat([a, b[rows]]) for a, b in
                          zip(y.rows[n], (values, y.new[:, L:].cpu().double())))
    cache = dict(rows=y.rows, lens=lens, dtype=BF16)
    want, wl, tol, ltol = ref.attention(cache, y.q, [D + 1] * N, y.scale)
    assert ref.close(y.out, want, tol) <= 1 and ref.close(y.lse, wl, ltol) <= 1
    host = {k: tuple(t.cpu() for t in v) if isinstance(v, tuple) else v.cpu()
            for k, v in y.s.items()}
    want = adjusted.definition(dict(host, logits=y.logits.cpu()))
    assert torch.equal(y.adjusted.cpu().double(), want)
    v = dict(target=y.adjusted, draft=y.draft, tokens=y.s["drafts"], accept_u=y.uniforms[0],
             sample_u=y.uniforms[1])
    accepted, tokens = verify.definition(v, False, False, 0.9)
    assert torch.equal(y.accepted.cpu(), accepted) and torch.equal(y.tokens.cpu(), tokens)


RESULTS = ("back", "out", "lse", "adjusted", "accepted", "tokens")


def fill(layer, seed):
    """Other inputs, and lengths that grow or fall, the first sequence's to none."""
    g = verify.gen(seed)
    for t in (layer.new, layer.q, layer.logits):
        t.copy_(torch.randn(t.shape, device=DEV, generator=g))
    lens = torch.randint(layer.D + 1, 600, (layer.N,), device=DEV, generator=g)
    lens[0] = 0 if seed % 2 else lens[0]
    layer.at.copy_(lens)


def same(a, b):
    assert torch.equal(a.cache["pool"], b.cache["pool"])
    for x in RESULTS:
        assert torch.equal(getattr(a, x), getattr(b, x)), x


def equal_layers(k3x, ctx, *args, **kw):
    """Two layers with buffers of their own that hold the same."""
    return tuple(Layer(k3x, ctx, *args, **kw) for _ in range(2))


@pytest.mark.parametrize("fmt", ["16bit", "mxfp8", "mxfp4"])
@pytest.mark.parametrize("H,D", [(4, 2), (32, 1), (64, 3)])
def test_captured_step(hip, fmt, H, D):
    """A step's calls in one graph; replays on changed inputs equal eager calls bit for bit."""
    k3x, _ = hip
    print(f"[gpu-test] captured step H={H} D={D} {fmt}", flush=True)
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        ctx = k3x.Context(0)
        one, two = equal_layers(k3x, ctx, [40, 3, 300], H, D, fmt, 3, more=600)
        for y in (one, two):
            fill(y, 2)
        one.step()
        two.step()
        assert ctx.synchronize() == 0
        graph = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, stream=stream):
            one.step()
        for i in range(4):
            for y in (one, two):
                fill(y, 10 + i)
            graph.replay()
            two.step()
            assert ctx.synchronize() == 0
            same(one, two)
        del graph
        ctx.close()


def test_captured_prompt(hip):
    """The same for a prompt's calls, its lengths read at each replay."""
    k3x, _ = hip
    H, T = 4, 700
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        ctx = k3x.Context(0)
        g = verify.gen(1)
        q, k, v = (torch.randn((T, H, d), device=DEV, generator=g).to(BF16)
                   for d in (192, 128, 128))
        rotary = torch.randn((T, 64), device=DEV, generator=g).to(BF16)
        outs = [torch.full((T, H, 128), -7.0, dtype=BF16, device=DEV) for _ in range(2)]
        offsets = mla.ints([0, 100, 100, 700])
        p = k3x.make_mla_prompt_params(q, k, v, 3, rotary=rotary, scale=0.07)

        def run(out):
            k3x.check(k3x.mla_prompt(ctx, p, q, k, v, out, rotary=rotary, offsets=offsets,
                                     key_offsets=offsets), "mla_prompt")
        run(outs[1])
        assert ctx.synchronize() == 0
        graph = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, stream=stream):
            run(outs[0])
        for i, cut in enumerate([[0, 100, 100, 700], [0, 0, 1, 400], [0, 333, 690, 700]]):
            offsets.copy_(mla.ints(cut))
            q.copy_(torch.randn(q.shape, device=DEV, generator=g))
            for out in outs:
                out.fill_(-7.0)
            graph.replay()
            run(outs[1])
            assert ctx.synchronize() == 0
            assert torch.equal(outs[0], outs[1]), i
            assert (outs[0][cut[-1]:] == -7).all() and (outs[0][:cut[-1]] != -7).any(-1).all()
        del graph
        ctx.close()


@pytest.mark.parametrize("fmt", ["16bit", "mxfp4"])
def test_two_streams(hip, fmt):
    """Two steps at once, each on a stream, context and workspace of its own, equal the same steps
    one after the other; the second pair of calls is a graph's replay beside an eager step."""
    k3x, ctx = hip
    H, D = 16, 3
    streams = [torch.cuda.Stream() for _ in range(2)]
    pairs, ctxs, graph = [], [], torch.cuda.CUDAGraph()
    for i, stream in enumerate(streams):
        with torch.cuda.stream(stream):
            ctxs.append(k3x.Context(0))
            pairs.append(equal_layers(k3x, ctxs[-1], [400, 90, 0, 7, 77], H, D, fmt, 3 + i,
                                      more=600))
            for y in pairs[-1]:
                fill(y, 20 + i)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=streams[0]):
        pairs[0][0].step()
    for i in range(4):
        for stream, pair in zip(streams, pairs):
            with torch.cuda.stream(stream):
                for y in pair:
                    fill(y, 30 + 2 * i)
        torch.cuda.synchronize()
        with torch.cuda.stream(streams[0]):
            graph.replay()
        with torch.cuda.stream(streams[1]):
            pairs[1][0].step()
        torch.cuda.synchronize()
        for stream, pair in zip(streams, pairs):
            with torch.cuda.stream(stream):
                pair[1].step()
            torch.cuda.synchronize()
        assert [c.synchronize() for c in ctxs] == [0, 0]
        for pair in pairs:
            same(*pair)
    del graph
    for c in ctxs:
        c.close()


def test_graphs_that_share_a_workspace(hip):
    """Calls with other numbers of sequences and heads, one after the other on one stream, keep
    nothing in a workspace for each other."""
    k3x, _ = hip
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        ctx = k3x.Context(0)
        a = equal_layers(k3x, ctx, [500, 20], 16, 1, "16bit", 1, more=600)
        b = equal_layers(k3x, ctx, [90] * 300, 4, 0, "16bit", 2, more=600)
        shared = torch.full((max(len(a[0].ws), len(b[0].ws)),), 255, dtype=torch.uint8, device=DEV)
        a[0].ws = b[0].ws = shared
        graphs = []
        torch.cuda.synchronize()
        for y in (a[0], b[0]):
            graphs.append(torch.cuda.CUDAGraph())
            with torch.cuda.graph(graphs[-1], stream=stream):
                y.store()
                y.attend()
        for i in range(4):
            for y in a + b:
                fill(y, 50 + i)
            for graph in (graphs if i % 2 else graphs[::-1]):
                graph.replay()
            for y in (a[1], b[1]):
                y.store()
                y.attend()
            assert ctx.synchronize() == 0
            for x, y in (a, b):
                assert torch.equal(x.out, y.out) and torch.equal(x.lse, y.lse)
        del graphs
        ctx.close()


@pytest.mark.parametrize("fmt", ["16bit", "mxfp8", "mxfp4"])
@pytest.mark.parametrize("H", [3, 29, 50, 64, 100, 300])
def test_rising_and_falling_scores(hip, fmt, H):
    """Largest scores that rise by hundreds within a tile and from tile to tile, each row's with a
    slope and a sign of its own, and rows whose largest is in one half of a tile's tokens."""
    k3x, ctx = hip
    n, wide = 3000, 256
    print(f"[gpu-test] rising scores H={H} {fmt}", flush=True)
    c = ref.make_cache([n, 130], wide, 0, 16, fmt, seed=H)
    g = ref.gen(H)
    for i, m in enumerate([n, 130]):
        rows = torch.randn((m, wide), generator=g)
        pos = torch.arange(m)
        rows[:, 0] = torch.linspace(-30, 30, m)
        rows[:, 1] = -torch.linspace(-20, 20, m).abs()
        rows[:, 2] = torch.where(pos // 32 % 2 == 1, 16.0, -16.0)
        none = torch.zeros((m, 0), dtype=BF16)
        data, values = ref.encode(rows.to(BF16), none, fmt)
        c["pool"][c["table"][i][pos // 16].long(), pos % 16] = data
        c["rows"][i] = (values, none.double())
    q = torch.randn((3, H, wide), generator=g) * 0.1
    q[..., :3] = torch.randn((3, H, 3), generator=g) * 8
    q = q.to(BF16)
    d = mla.to_device(c)
    p = mla.params(k3x, d, 3, H, 1.0, longest=2)
    out = torch.empty((3, H, wide), dtype=BF16, device=DEV)
    lse = torch.empty((3, H), device=DEV)
    ws = torch.empty((k3x.mla_attention_workspace_bytes(p),), dtype=torch.uint8, device=DEV)
    assert k3x.mla_attention(ctx, p, q.to(DEV), d["pool"], d["table"], mla.ints([n, 130]), out,
                             offsets=mla.offsets_of([1, 2]), lse=lse, workspace=ws) == 0
    assert ctx.synchronize() == 0
    want, wl, tol, ltol = ref.attention(c, q, [1, 2], 1.0)
    assert ref.close(out, want, tol) <= 1 and ref.close(lse, wl, ltol) <= 1


@pytest.mark.parametrize("fmt", ["16bit", "mxfp8", "mxfp4"])
@pytest.mark.parametrize("norm", [True, False], ids=["norm", "plain"])
def test_many_tokens(hip, fmt, norm):
    """More tokens than waves take one by one, with empty sequences, ones padded to the left, first rows that
    are no sequence's and rows past the last."""
    k3x, ctx = hip
    counts = [0, 0, 3, 8200, 0, 1] + [1] * 75 + [0] * 70 + [8200, 0, 9, 17]
    lens = [5, 0, 2, 8200, 9, 1] + [3] * 75 + [0] * 70 + [8300, 1, 9, 10]
    first, spare, page = 5, 30, 64
    T = first + sum(counts) + spare
    assert T > 16384
    print(f"[gpu-test] {T} tokens {fmt}", flush=True)
    g = ref.gen(8)
    c = ref.make_cache(lens, L, R, page, fmt, seed=4)
    x = torch.randn((T, L + R), generator=g).to(BF16)
    gamma = 1 + 0.2 * torch.randn(L, generator=g)
    offsets = [first + sum(counts[:i]) for i in range(len(counts) + 1)]
    d = mla.to_device(c)
    p = mla.params(k3x, d, T, eps=EPS)
    xd = x.to(DEV)
    assert k3x.mla_store(ctx, p, xd[:, :L], d["pool"], d["table"], mla.ints(lens),
                         rotary=xd[:, L:], offsets=mla.ints(offsets),
                         gamma=gamma.to(DEV) if norm else None) == 0
    back = torch.full((T, L), 7.0, dtype=BF16, device=DEV)
    turned = torch.full((T, R), 7.0, dtype=BF16, device=DEV)
    assert k3x.mla_load(ctx, p, d["pool"], d["table"], mla.ints(lens), back, rotary=turned,
                        offsets=mla.ints(offsets)) == 0
    assert ctx.synchronize() == 0
    y = x[:, :L]
    if norm:
        z = y.double()
        y = (z / torch.sqrt((z * z).mean(-1, keepdim=True) + F32_EPS) *
             gamma.double()).float().to(BF16)
    data, values = ref.encode(y, x[:, L:], fmt)
    want, hold = c["pool"].clone(), torch.full((T, L), 7.0, dtype=torch.float64)
    turn = torch.full((T, R), 7.0, dtype=torch.float64)
    for n, m in enumerate(counts):
        t = torch.arange(offsets[n], offsets[n + 1])
        pos = lens[n] - m + torch.arange(m)
        t, pos = t[pos >= 0], pos[pos >= 0]
        want[c["table"][n, pos // page].long(), pos % page] = data[t]
        hold[t], turn[t] = values[t], x[t, L:].double()
    assert torch.equal(d["pool"].cpu(), want)
    assert torch.equal(back.cpu().double(), hold) and torch.equal(turned.cpu().double(), turn)


def test_no_tokens(hip):
    """Calls of no tokens write nothing; queries without a key have zeros."""
    k3x, ctx = hip
    c = mla.to_device(ref.make_cache([4, 9], L, R, 16))
    before = c["pool"].clone()
    p = mla.params(k3x, c, 0, 4)
    empty = torch.empty((0, L), dtype=BF16, device=DEV)
    q, out = (torch.empty((0, 4, d), dtype=BF16, device=DEV) for d in (L + R, L))
    ws = torch.empty((k3x.mla_attention_workspace_bytes(p),), dtype=torch.uint8, device=DEV)
    args = (c["pool"], c["table"], mla.ints([4, 9]))
    for offsets in (None, mla.ints([0, 0, 0])):
        assert k3x.mla_store(ctx, p, empty, *args, rotary=empty[:, :R], offsets=offsets) == 0
        assert k3x.mla_load(ctx, p, *args, empty, offsets=offsets) == 0
        assert k3x.mla_attention(ctx, p, q, *args, out, offsets=offsets, workspace=ws) == 0
    assert ctx.synchronize() == 0
    assert torch.equal(c["pool"], before)
    k, rotary = q[..., :64], empty[:, :R]
    for T in (0, 6):
        qs = torch.ones((T, 4, 64 + R), dtype=BF16, device=DEV)
        outs = torch.full((T, 4, 64), 7.0, dtype=BF16, device=DEV)
        lse = torch.full((T, 4), 7.0, device=DEV)
        for rot in (rotary, None):
            x = qs if rot is not None else qs[..., :64].contiguous()
            pp = k3x.make_mla_prompt_params(x, k, k, 2, rotary=rot)
            assert k3x.mla_prompt(ctx, pp, x, k, k, outs, rotary=rot, lse=lse) == 0
        assert ctx.synchronize() == 0
        assert (outs == 0).all() and (lse == -torch.inf).all()
