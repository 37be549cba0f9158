"""The adjustment of logits beside sequences that are not fit, and of rows past 32-bit offsets."""
from __future__ import annotations

import pytest

import test_gpu_logits as base

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


def many(N, D, V, dtype):
    """Inputs of many sequences on the device, each with a history of 30 tokens."""
    g = torch.Generator(device=DEV)
    g.manual_seed(N + V)

    def ints(hi, *shape):
        return torch.randint(0, hi, shape, device=DEV, generator=g).int()
    return dict(logits=torch.randn((N, D + 1, V), device=DEV, generator=g).to(dtype),
                history=ints(V, N, 30), history_lens=torch.full((N,), 30, device=DEV).int(),
                drafts=ints(V, N, D), masks=ints(1 << 30, 3, -(-V // 32)),
                mask_index=ints(3, N, D + 1),
                repetition=torch.full((N,), 1.3, device=DEV),
                frequency=torch.full((N,), 0.2, device=DEV))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("what", ["history", "token", "draft", "repetition"])
def test_an_unfit_sequence_leaves_the_others_whole(hip, dtype, what):
    """In place a call cannot be repeated: all rows of the other sequences are adjusted, those of
    workgroups that begin after the error was found too.  More workgroups than begin at once."""
    k3x, ctx = hip
    N, D, V = 300, 1, 50001
    s = many(N, D, V, dtype)
    x = s.pop("logits")
    p = k3x.make_logits_params(x)
    want = torch.empty_like(x)
    assert k3x.adjust_logits(ctx, p, x, want, **s) == 0
    assert ctx.synchronize() == 0
    bad = 0
    if what == "history":
        s["history_lens"][bad] = 31
    elif what == "token":
        s["history"][bad, 3] = V
    elif what == "draft":
        s["drafts"][bad, 0] = V
    else:
        s["repetition"][bad] = -1.0
    print(f"[gpu-test] logits in place beside unfit {what}", flush=True)
    for _ in range(3):
        y = x.clone()
        assert k3x.adjust_logits(ctx, p, y, y, **s) == 0
        assert ctx.synchronize() == k3x.ERR_INVALID_STATE
        assert torch.equal(y[1:], want[1:])
        # And nothing of the error is left for the next call.
        y = x.clone()
        t = {k: v[1:].contiguous() if k not in ("masks",) else v for k, v in s.items()}
        assert k3x.adjust_logits(ctx, k3x.make_logits_params(y[1:]), y[1:], y[1:], **t) == 0
        assert ctx.synchronize() == 0
        assert torch.equal(y[1:], want[1:]) and torch.equal(y[0], x[0])


def test_captured_calls_beside_an_unfit_sequence(hip):
    """In place, replayed with an unfit sequence in one replay."""
    k3x, _ = hip
    N, D, V = 40, 2, 20011
    s = many(N, D, V, torch.bfloat16)
    x = s.pop("logits")
    stream = torch.cuda.Stream()
    print("[gpu-test] captured logits beside an unfit sequence", flush=True)
    with torch.cuda.stream(stream):
        ctx = k3x.Context(0)
        p = k3x.make_logits_params(x)
        want, y = torch.empty_like(x), x.clone()
        assert k3x.adjust_logits(ctx, p, x, want, **s) == 0
        assert ctx.synchronize() == 0
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            assert k3x.adjust_logits(ctx, p, y, y, **s) == 0
    for i in range(5):
        y.copy_(x)
        s["history_lens"][5] = 31 if i % 2 else 30
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert ctx.synchronize() == (k3x.ERR_INVALID_STATE if i % 2 else 0)
        left = [n for n in range(N) if n != 5 or not i % 2]
        assert torch.equal(y[left], want[left])
    ctx.close()


@pytest.mark.parametrize("in_place", [False, True], ids=["out", "in_place"])
def test_rows_past_32_bit_offsets(hip, in_place):
    """Rows 2^31 elements apart."""
    k3x, ctx = hip
    s = base.make(2, 1, 5001, torch.bfloat16)
    wide = torch.empty((4, (1 << 31) + 8), dtype=torch.bfloat16, device=DEV)
    x = wide[:, :5001].unflatten(0, (2, 2))
    x.copy_(s["logits"].to(DEV))
    out = x if in_place else wide[:, 8192:8192 + 5001].unflatten(0, (2, 2))
    d = {k: tuple(t.to(DEV) for t in v) if isinstance(v, tuple) else v.to(DEV)
         for k, v in s.items() if k != "logits"}
    print("[gpu-test] logits 2^31 elements apart", flush=True)
    assert k3x.adjust_logits(ctx, k3x.make_logits_params(x), x, out, **d) == 0
    assert ctx.synchronize() == 0
    assert torch.equal(out.double().cpu(), base.definition(s))
