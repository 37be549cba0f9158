"""Attention of prompts over expanded keys and values (k3x_hip_mla_prompt) against a plain
implementation in 64 bits, within the tolerance that mla_reference.softmax_rows derives."""
from __future__ import annotations

import math

import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")
import mla_reference as ref  # noqa: E402

DEV = "cuda:0"
BF16, F16 = torch.bfloat16, torch.float16


@pytest.fixture(scope="module")
def hip():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    import k3x_amd
    ctx = k3x_amd.Context(0)
    yield k3x_amd, ctx
    ctx.close()


def say(text):
    print(f"[gpu-test] {text}", flush=True)


def offsets_of(counts):
    return torch.tensor([sum(counts[:i]) for i in range(len(counts) + 1)], dtype=torch.int32,
                        device=DEV)


def inputs(counts, keys, H, Dn, R, Dv, dtype, seed=0, spread=1.0, extra=0):
    """k and v as parts of one projection's rows; rows past the last sequence are NaN."""
    g = ref.gen(seed + 31 * H + Dn)
    T, S = sum(counts), sum(keys)
    q = (torch.randn((T + extra, H, Dn + R), generator=g) * spread).to(dtype)
    kv = torch.randn((S + extra, H, Dn + Dv), generator=g).to(dtype)
    rotary = torch.randn((S + extra, R), generator=g).to(dtype) if R else None
    if extra:
        kv[S:] = math.nan
        if R:
            rotary[S:] = math.nan
    return q, kv, rotary


def case(hip, counts, keys, H=2, Dn=128, R=64, Dv=128, dtype=BF16, causal=True, scale=None,
         seed=0, spread=1.0, extra=0, offsets=True, longest=None):
    k3x, ctx = hip
    say(f"prompt {counts} over {keys} H={H} {Dn}+{R}/{Dv} {dtype} causal={causal} extra={extra}")
    scale = float(torch.tensor((Dn + R) ** -0.5 if scale is None else scale))
    q, kv, rotary = inputs(counts, keys, H, Dn, R, Dv, dtype, seed, spread, extra)
    T = sum(counts)
    qd, kvd = q.to(DEV), kv.to(DEV)
    rd = rotary.to(DEV) if R else None
    k, v = kvd[..., :Dn], kvd[..., Dn:]
    out = torch.full((T + extra, H, Dv), 7.0, dtype=dtype, device=DEV)
    lse = torch.full((T + extra, H), 7.0, device=DEV)
    p = k3x.make_mla_prompt_params(qd, k, v, len(counts), rotary=rd, causal=causal, scale=scale,
                                   longest=max(counts) if longest is None else longest)
    st = k3x.mla_prompt(ctx, p, qd, k, v, out, rotary=rd,
                        offsets=offsets_of(counts) if offsets else None,
                        key_offsets=offsets_of(keys) if offsets else None, lse=lse)
    assert (st, ctx.synchronize()) == (0, 0)
    want, wl, tol, ltol = ref.prompt(q, kv[..., :Dn], kv[..., Dn:], rotary, counts, keys, causal,
                                     scale)
    assert (out[T:] == 7).all() and (lse[T:] == 7).all()
    a, b = ref.close(out[:T], want[:T], tol[:T]), ref.close(lse[:T], wl[:T], ltol[:T])
    assert a <= 1 and b <= 1, (a, b)


@pytest.mark.parametrize("dtype", [BF16, F16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("causal", [True, False], ids=["causal", "all"])
@pytest.mark.parametrize("counts,keys", [
    ([1], [1]), ([33], [33]), ([128], [128]), ([129], [129]), ([5, 0, 64, 1], [5, 7, 70, 200]),
    ([31, 257], [32, 300]), ([40, 3], [0, 2]), ([10], [4])], ids=str)
def test_lengths(hip, dtype, causal, counts, keys):
    """Prefixes, sequences without queries or keys, queries that see nothing."""
    case(hip, counts, keys, dtype=dtype, causal=causal)


@pytest.mark.parametrize("dtype", [BF16, F16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("Dn,R,Dv", [(128, 64, 128), (128, 0, 128), (64, 32, 64), (72, 24, 104),
                                     (32, 0, 40), (8, 8, 8), (120, 56, 16), (16, 64, 120),
                                     (64, 64, 64), (96, 0, 128)])
def test_widths(hip, dtype, Dn, R, Dv):
    case(hip, [70, 9], [100, 9], 3, Dn, R, Dv, dtype)


@pytest.mark.parametrize("H", [1, 5, 16])
def test_heads(hip, H):
    case(hip, [65, 30], [65, 131], H)


def test_long(hip):
    case(hip, [600], [600], 1)
    case(hip, [3, 200], [1500, 900], 1)


@pytest.mark.parametrize("dtype", [BF16, F16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("Dn,R", [(128, 64), (128, 0), (64, 64)])
def test_many_rows(hip, dtype, Dn, R):
    """More workgroups than begin at once."""
    case(hip, [300, 1, 0, 257, 40, 140], [300, 77, 5, 400, 39, 140], 256, Dn, R, 128, dtype)
    case(hip, [1100], [1300], 128, Dn, R, 128, dtype, causal=False)


def test_many_sequences(hip):
    counts = [n % 5 for n in range(150)]
    case(hip, counts, [c + n % 7 for n, c in enumerate(counts)], 2, 64, 32, 64)


@pytest.mark.parametrize("causal", [True, False], ids=["causal", "all"])
@pytest.mark.parametrize("N", [2, 63, 64, 65])
@pytest.mark.parametrize("hint", [None, 5000])
def test_order_of_blocks(hip, N, causal, hint):
    """Each block of queries is taken once, however lengths order them: one long sequence, many
    equal ones, more queries than keys and none."""
    g = ref.gen(N)
    counts = torch.randint(0, 300, (N,), generator=g).tolist()
    keys = [c + int(k) for c, k in zip(counts, torch.randint(-40, 200, (N,), generator=g))]
    counts[0], keys[0], keys[1] = 1400, 1500, 0
    case(hip, counts, [max(0, k) for k in keys], 1, 64, 0, 64, causal=causal, longest=hint)
    case(hip, [130] * N, [200] * N, 1, 64, 0, 64, causal=causal, longest=hint)


def test_without_offsets(hip):
    case(hip, [20, 20, 20], [30, 30, 30], offsets=False)


@pytest.mark.parametrize("longest", [0, 1, 1000])
def test_longest_is_a_hint(hip, longest):
    case(hip, [150, 20], [150, 40], longest=longest)


def test_rows_past_the_last_sequence(hip):
    case(hip, [40, 33], [50, 33], extra=5)


def test_sharp_and_flat_scores(hip):
    case(hip, [90], [200], spread=15.0)
    case(hip, [90], [200], scale=1e-4)


def test_layouts(hip):
    """Heads outermost, packed rows, one head of a wider row."""
    k3x, ctx = hip
    T, H, Dn, Dv = 45, 3, 64, 64
    g = ref.gen(4)
    q = torch.randn((T, H, Dn), generator=g).to(BF16)
    k = torch.randn((H, T, Dn), generator=g).to(BF16)
    v = torch.randn((T, H, Dv), generator=g).to(BF16)
    kd = k.to(DEV).transpose(0, 1)
    wide = torch.zeros((T, H * Dv + 8), dtype=BF16, device=DEV)
    out = wide[:, :H * Dv].view(T, H, Dv)
    p = k3x.make_mla_prompt_params(q.to(DEV), kd, v.to(DEV), 1, scale=0.125)
    say("prompt layouts")
    assert k3x.mla_prompt(ctx, p, q.to(DEV), kd, v.to(DEV), out) == 0
    assert ctx.synchronize() == 0
    want, _, tol, _ = ref.prompt(q, k.transpose(0, 1), v, None, [T], [T], True, 0.125)
    assert ref.close(out, want, tol) <= 1
    assert (wide[:, H * Dv:] == 0).all()


@pytest.mark.parametrize("where", ["q", "k", "v", "rotary"])
def test_values_that_are_not_finite_are_latched(hip, where):
    k3x, ctx = hip
    q, kv, rotary = (x.to(DEV) for x in inputs([40], [40], 2, 64, 16, 64, BF16))
    t = {"q": q[30, 1], "k": kv[30, 1, :64], "v": kv[30, 1, 64:], "rotary": rotary[30]}[where]
    t[5] = math.nan
    out = torch.zeros((40, 2, 64), dtype=BF16, device=DEV)
    p = k3x.make_mla_prompt_params(q, kv[..., :64], kv[..., 64:], 1, rotary=rotary, scale=0.1)
    say(f"prompt with NaN in {where}")
    assert k3x.mla_prompt(ctx, p, q, kv[..., :64], kv[..., 64:], out, rotary=rotary) == 0
    assert ctx.synchronize() == k3x.ERR_INVALID_MXFP4
    assert ctx.synchronize() == 0


@pytest.mark.parametrize("which", ["q falls", "q past", "k falls", "k past"])
def test_unfit_offsets_are_latched(hip, which):
    k3x, ctx = hip
    q, kv, rotary = (x.to(DEV) for x in inputs([20, 20], [30, 30], 2, 64, 16, 64, BF16))
    qo, ko = offsets_of([20, 20]), offsets_of([30, 30])
    if which == "q falls":
        qo[1] = 41
    elif which == "q past":
        qo[2] = 41
    elif which == "k falls":
        ko[1] = 61
    else:
        ko[2] = 61
    guard = torch.full((42, 2, 64), 7.0, dtype=BF16, device=DEV)
    p = k3x.make_mla_prompt_params(q, kv[..., :64], kv[..., 64:], 2, rotary=rotary, scale=0.1)
    say(f"prompt: {which}")
    assert k3x.mla_prompt(ctx, p, q, kv[..., :64], kv[..., 64:], guard[1:41], rotary=rotary,
                          offsets=qo, key_offsets=ko) == 0
    assert ctx.synchronize() == k3x.ERR_INVALID_STATE
    assert (guard[0] == 7).all() and (guard[41] == 7).all()
    assert ctx.synchronize() == 0
