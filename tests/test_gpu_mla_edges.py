"""Latent attention where it can go wrong silently: scores that are no numbers, small weights
beside a large one, values at the end of their type, calls of no tokens, the most that a call
takes, distances past 32 bits, and largest scores that rise within a range in every layout."""
from __future__ import annotations

import math

import pytest

import mla_reference as ref
import test_gpu_mla as mla

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")
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


def plain_cache(lens, L, R, page, latent, rotary, dtype=BF16):
    """A 16-bit cache of one row for every position: latent [n][L] and rotary [n][R] of the longest
    sequence, of which the others have the first rows."""
    counts = [-(-n // page) for n in lens]
    width = max(counts)
    n = max(lens)
    data = ref.encode(latent.to(dtype), rotary.to(dtype), "16bit")[0]
    pool = torch.zeros((width * page, data.shape[1]), dtype=torch.uint8)
    pool[:n] = data
    table = torch.arange(width, dtype=torch.int32).repeat(len(lens), 1)
    return dict(pool=pool.view(width, page, -1).to(DEV), table=table.to(DEV), L=L, R=R,
                fmt="16bit", dtype=dtype)


def attend(hip, c, q, lens, scale=1.0, longest=1, offsets=None):
    """(status that was latched, out, lse); workspace and outputs full of other bytes."""
    k3x, ctx = hip
    T, H = q.shape[:2]
    p = mla.params(k3x, c, T, H, scale, longest=longest)
    out = torch.full((T, H, c["L"]), 7.0, dtype=c["dtype"], device=DEV)
    lse = torch.full((T, H), 7.0, device=DEV)
    ws = torch.full((k3x.mla_attention_workspace_bytes(p),), 255, dtype=torch.uint8, device=DEV)
    assert k3x.mla_attention(ctx, p, q.to(DEV), c["pool"], c["table"], mla.ints(lens), out,
                             offsets=offsets, lse=lse, workspace=ws) == 0
    return ctx.synchronize(), out.double().cpu(), lse.double().cpu()


def prompt(hip, q, k, v, rotary, scale=1.0, causal=True, **kw):
    k3x, ctx = hip
    q, k, v = q.to(DEV), k.to(DEV), v.to(DEV)
    rotary = None if rotary is None else rotary.to(DEV)
    out = torch.full((q.shape[0], q.shape[1], v.shape[2]), 7.0, dtype=q.dtype, device=DEV)
    lse = torch.full(q.shape[:2], 7.0, device=DEV)
    p = k3x.make_mla_prompt_params(q, k, v, 1, rotary=rotary, causal=causal, scale=scale)
    assert k3x.mla_prompt(ctx, p, q, k, v, out, rotary=rotary, lse=lse, **kw) == 0
    return ctx.synchronize(), out.double().cpu(), lse.double().cpu()


def long_calls(hip, counts, lens, H, longest, L=32):
    """Attention over one page of equal rows that every position of every sequence is in."""
    page, width = 65536, 8192
    N = len(lens)
    data = ref.encode(torch.ones((1, L), dtype=BF16), torch.zeros((1, 0), dtype=BF16), "16bit")[0]
    c = dict(pool=data.repeat(page, 1).view(1, page, -1).to(DEV),
             table=torch.zeros((N, width), dtype=torch.int32, device=DEV), L=L, R=0, fmt="16bit",
             dtype=BF16)
    q = torch.ones((sum(counts), H, L), dtype=BF16)
    mla.say(f"{N} sequences, longest {max(lens)}, {H} heads")
    return attend(hip, c, q, lens, 1.0, longest, mla.offsets_of(counts))


def test_most_rows_of_the_longest_sequence(hip):
    """128 rows over 2^29 positions, in blocks of 64 beside single tokens."""
    n = 1 << 29
    st, out, lse = long_calls(hip, [2] + [1] * 31 + [0] * 32, [n] + [1] * 31 + [0] * 32, 64, 16)
    assert st == 0
    assert (out == 1).all()
    sees = torch.tensor([n - 1, n] + [1] * 31, dtype=torch.float64)
    # Equal weights: sums of ones up to 2^21 a range, exact, and their 256 pieces.
    assert float((lse - 32 - sees.log()[:, None]).abs().max()) <= 2.0 ** -17


@pytest.mark.parametrize("total", [1 << 31, (1 << 31) + 5, (1 << 32) - 600, (1 << 32) - 100,
                                   (1 << 32) - 1, 1 << 32, (1 << 32) + 70], ids=hex)
def test_more_than_a_call_takes_is_latched(hip, total):
    """Sequences that make 2^31 tiles of 32 positions together and more, around what 32 bits hold:
    latched before a page is looked at."""
    k3x, ctx = hip
    each, lens = 1 << 24, []
    while total:
        lens.append(min(each, total) * 32)
        total -= min(each, total)
    st, _, _ = long_calls(hip, [1] * len(lens), lens, 1, 1)
    assert st == k3x.ERR_INVALID_STATE
    assert ctx.synchronize() == 0


# Rows a block and layouts: heads, latent, rotary part.
LAYOUTS = [(4, 512, 64), (24, 512, 64), (48, 512, 64), (96, 512, 64), (4, 96, 16), (48, 96, 16)]


@pytest.mark.parametrize("H,L,R", LAYOUTS)
@pytest.mark.parametrize("n", [1, 20, 4000])
@pytest.mark.parametrize("finite", [False, True], ids=["infinity", "overflow"])
def test_scores_of_minus_infinity_are_latched(hip, H, L, R, n, finite):
    """A row whose scores are all minus infinity has no softmax: it is not one that sees nothing."""
    k3x, ctx = hip
    mla.say(f"scores of minus infinity H={H} L={L} n={n} finite={finite}")
    rotary = torch.zeros((n, R))
    rotary[:, 3] = 3e38 if finite else 1.0
    c = plain_cache([n, n], L, R, 16, torch.ones((n, L)), rotary)
    q = torch.ones((2, H, L + R), dtype=BF16)
    q[:, :, L + 3] = 0
    q[1, H - 1, L + 3] = -3e38 if finite else -math.inf
    st, out, lse = attend(hip, c, q, [n, n], 2.0 ** -20)
    assert st == k3x.ERR_INVALID_MXFP4
    assert ctx.synchronize() == 0
    # Without that row nothing is latched, and a token that sees nothing has zeros.
    q[1, H - 1, L + 3] = 0
    st, out, lse = attend(hip, c, q, [n, 0], 2.0 ** -20)
    assert st == 0
    assert (out[0] == 1).all() and (out[1] == 0).all() and (lse[1] == -math.inf).all()


@pytest.mark.parametrize("Dn,R", [(128, 64), (128, 0), (64, 16)])
@pytest.mark.parametrize("m,n", [(1, 1), (70, 300), (40, 3)])
@pytest.mark.parametrize("causal", [True, False], ids=["causal", "all"])
def test_prompt_scores_of_minus_infinity_are_latched(hip, Dn, R, m, n, causal):
    k3x, ctx = hip
    mla.say(f"prompt scores of minus infinity {Dn}+{R} {m} over {n}")
    q = torch.ones((m, 2, Dn + R), dtype=BF16)
    k, v = torch.ones((n, 2, Dn), dtype=BF16), torch.ones((n, 2, 64), dtype=BF16)
    rotary = torch.ones((n, R), dtype=BF16) if R else None
    st, out, lse = prompt(hip, q, k, v, rotary, 0.1, causal)
    assert st == 0
    none = max(0, m - n) if causal else 0  # queries that see nothing
    assert (out[none:] == 1).all() and (out[:none] == 0).all()
    assert (lse[:none] == -math.inf).all()
    q[m - 1, 1, 5] = -math.inf
    st, out, lse = prompt(hip, q, k, v, rotary, 0.1, causal)
    assert st == k3x.ERR_INVALID_MXFP4
    assert ctx.synchronize() == 0


# What many equal weights beside a large one are off by, all values 1.  A weight is rounded by
# half a step of fp16, 2^-11 of it or (below 2^-14) 2^-25; the row's largest is 2^7 at least, so
# that n weights miss n 2^-32 of the sum.  The sums of weights and of outputs are `adds` fp32
# additions in a row (the matrix cores may cut where they do not round: 2^-23 each), the
# exponentials 2^-20, and the output is rounded by 2^-11.
def small_weights_tolerance(n, adds):
    return 2 * 2.0 ** -11 + n * 2.0 ** -32 + adds * 2.0 ** -23 + 2.0 ** -20


@pytest.mark.parametrize("N,H,L,R", [(512, 1, 512, 64), (256, 24, 512, 64), (256, 48, 512, 64),
                                     (256, 96, 512, 64), (512, 1, 96, 16), (256, 48, 96, 16)])
def test_small_weights_in_fp16(hip, N, H, L, R):
    """Weights just below 2^-25 of the largest one: alone they are nothing, together 0.3%.  So many
    sequences (of the same pages) that each lies in one range or two."""
    n = 100001
    mla.say(f"small weights N={N} H={H} L={L}")
    rotary = torch.zeros((n, R))
    rotary[0, 0] = 1
    c = plain_cache([n] * N, L, R, 64, torch.ones((n, L)), rotary, F16)
    q = torch.zeros((N, H, L + R), dtype=F16)
    q[:, :, L] = 1
    scale = 25.05 * math.log(2)
    st, out, lse = attend(hip, c, q, [n] * N, scale)
    assert st == 0
    rest = (n - 1) * 2.0 ** -25.05
    # 16 tokens a product at least: 6251 additions to an output, fewer to a sum.
    assert rest > small_weights_tolerance(n, 6400)
    assert float((out - 1).abs().max()) <= small_weights_tolerance(n, 6400)
    assert float((lse - scale - math.log1p(rest)).abs().max()) <= 2.0 ** -9


@pytest.mark.parametrize("Dn,R", [(128, 64), (64, 16)])
def test_small_weights_in_fp16_prompts(hip, Dn, R):
    n, m = 80000, 3
    mla.say(f"small weights of a prompt {Dn}+{R}")
    rotary = torch.zeros((n, R), dtype=F16)
    rotary[0, 0] = 1
    q = torch.zeros((m, 1, Dn + R), dtype=F16)
    q[:, :, Dn] = 1
    k, v = torch.zeros((n, 1, Dn), dtype=F16), torch.ones((n, 1, 64), dtype=F16)
    scale = 25.05 * math.log(2)
    st, out, lse = prompt(hip, q, k, v, rotary, scale)
    assert st == 0
    rest = (n - m) * 2.0 ** -25.05
    # 16 keys a product: 5000 additions to an output, fewer to a sum.
    assert rest > small_weights_tolerance(n, 5100)
    assert float((out - 1).abs().max()) <= small_weights_tolerance(n, 5100)
    assert float((lse - scale - math.log1p(rest)).abs().max()) <= 2.0 ** -9


@pytest.mark.parametrize("H,L,R", [(1, 512, 64), (24, 512, 64), (48, 512, 64), (96, 512, 64),
                                   (1, 96, 16), (48, 96, 16)])
@pytest.mark.parametrize("n", [40, 2001])
@pytest.mark.parametrize("sign", [1, -1])
def test_largest_values_of_fp16(hip, H, L, R, n, sign):
    """Outputs are between the values, also where all weights but the largest round up and their
    sum does not: 65504 times that passes what fp16 holds."""
    mla.say(f"largest values H={H} L={L} n={n}")
    rotary = torch.full((n, R), -1.0)
    rotary[0] = 0
    c = plain_cache([n], L, R, 16, torch.full((n, L), sign * 65504.0), rotary, F16)
    q = torch.zeros((1, H, L + R), dtype=F16)
    q[:, :, L] = 1
    st, out, _ = attend(hip, c, q, [n], -math.log((1 + 2.0 ** -11 + 2.0 ** -13) / 2))
    assert st == 0 and (out == sign * 65504).all()


@pytest.mark.parametrize("Dn,R", [(128, 64), (64, 16)])
def test_largest_values_of_fp16_in_prompts(hip, Dn, R):
    n = 200
    rotary = torch.full((n, R), -1.0, dtype=F16)
    rotary[0] = 0
    q = torch.zeros((n, 1, Dn + R), dtype=F16)
    q[:, :, Dn] = 1
    k, v = torch.zeros((n, 1, Dn), dtype=F16), torch.full((n, 1, 64), 65504.0, dtype=F16)
    mla.say(f"largest values of a prompt {Dn}+{R}")
    st, out, _ = prompt(hip, q, k, v, rotary, -math.log((1 + 2.0 ** -11 + 2.0 ** -13) / 2))
    assert st == 0 and (out == 65504).all()


@pytest.mark.parametrize("H", [1, 24, 48, 96])
def test_sums_past_fp32_are_latched(hip, H):
    """Pieces of a sequence that are numbers each, and whose sum is not."""
    k3x, ctx = hip
    n = 60000
    mla.say(f"sums past fp32 H={H}")
    c = plain_cache([n], 512, 64, 64, torch.full((n, 512), 1e35), torch.zeros((n, 64)))
    q = torch.zeros((1, H, 576), dtype=BF16)
    st, out, _ = attend(hip, c, q, [n])
    assert st == k3x.ERR_INVALID_MXFP4
    assert ctx.synchronize() == 0


# Scores of 3.6e9 times this: their rounded product with log2(e) is 82 off, so that in fp32 the
# largest weight is 2^-82, and its sum a number; in fp16 it is nothing.
FAR = 1.01


@pytest.mark.parametrize("H,L,R", [(1, 512, 64), (24, 512, 64), (48, 512, 64), (96, 512, 64),
                                   (1, 96, 16), (48, 96, 16)])
@pytest.mark.parametrize("n", [1, 2001])
def test_scores_past_fp16_weights_are_latched(hip, H, L, R, n):
    k3x, ctx = hip
    mla.say(f"scores of 3.6e9 H={H} L={L} n={n}")
    for dtype, want in ((F16, k3x.ERR_INVALID_MXFP4), (BF16, 0)):
        # 60000 in fp16, in bf16 59904.
        c = plain_cache([n], L, R, 16, torch.ones((n, L)), torch.full((n, R), 60000.0), dtype)
        q = torch.zeros((1, H, L + R), dtype=dtype)
        q[:, :, L] = 60000
        st, out, _ = attend(hip, c, q, [n], FAR)
        assert st == want
        assert ctx.synchronize() == 0
        if not want:
            assert (out == 1).all()


@pytest.mark.parametrize("Dn,R", [(128, 64), (64, 16)])
def test_prompt_scores_past_fp16_weights_are_latched(hip, Dn, R):
    k3x, ctx = hip
    mla.say(f"prompt scores of 3.6e9 {Dn}+{R}")
    rotary = torch.full((40, R), 60000.0, dtype=F16)
    q = torch.zeros((5, 1, Dn + R), dtype=F16)
    q[:, :, Dn] = 60000
    k, v = torch.zeros((40, 1, Dn), dtype=F16), torch.ones((40, 1, 64), dtype=F16)
    st, _, _ = prompt(hip, q, k, v, rotary, FAR)
    assert st == k3x.ERR_INVALID_MXFP4
    assert ctx.synchronize() == 0


@pytest.mark.parametrize("what", ["offsets", "length", "keys"])
def test_calls_of_no_tokens_are_checked(hip, what):
    """Offsets and lengths are looked at in calls of no tokens too, by every call."""
    k3x, ctx = hip
    c = mla.to_device(ref.make_cache([4, 9], 64, 16, 16))
    p = mla.params(k3x, c, 0, 4)
    lens = mla.ints([4, 17 if what == "length" else 9])
    offsets = mla.ints([0, 1, 1] if what == "offsets" else [0, 0, 0])
    q, out = (torch.empty((0, 4, d), dtype=BF16, device=DEV) for d in (80, 64))
    latent = torch.empty((0, 64), dtype=BF16, device=DEV)
    ws = torch.empty((k3x.mla_attention_workspace_bytes(p),), dtype=torch.uint8, device=DEV)
    k = torch.zeros((6, 4, 64), dtype=BF16, device=DEV)
    pp = k3x.make_mla_prompt_params(q[..., :64].contiguous(), k, k, 2)
    calls = [lambda: k3x.mla_prompt(ctx, pp, q[..., :64].contiguous(), k, k, out, offsets=offsets,
                                    key_offsets=mla.ints([0, 7, 7] if what == "keys" else
                                                         [0, 3, 6]))]
    if what != "keys":
        calls += [lambda: k3x.mla_attention(ctx, p, q, c["pool"], c["table"], lens, out,
                                            offsets=offsets, workspace=ws),
                  lambda: k3x.mla_store(ctx, p, latent, c["pool"], c["table"], lens,
                                        rotary=latent[:, :16], offsets=offsets),
                  lambda: k3x.mla_load(ctx, p, c["pool"], c["table"], lens, latent,
                                       offsets=offsets)]
    if what == "length":
        calls = calls[1:]
    for i, call in enumerate(calls):
        mla.say(f"no tokens, unfit {what}, call {i}")
        assert call() == 0
        assert ctx.synchronize() == k3x.ERR_INVALID_STATE
        assert ctx.synchronize() == 0


@pytest.mark.parametrize("m", [1, 5])
def test_prompt_over_one_key_of_a_cache(hip, m):
    """One key of a cache whose heads lie far apart: rows of it have no distance."""
    k3x, ctx = hip
    H, D, most = 9, 64, (1 << 18) + 8
    g = ref.gen(m)
    store = torch.zeros((H, most, D), dtype=BF16, device=DEV)
    kv = torch.randn((1, H, D), generator=g).to(BF16)
    store[:, 0] = kv[0].to(DEV)
    k = store[:, :1].transpose(0, 1)
    q = torch.randn((m, H, D), generator=g).to(BF16)
    mla.say(f"prompt of {m} over one key")
    st, out, lse = prompt(hip, q, k, k, None, 0.125)
    assert st == 0
    want, wl, tol, ltol = ref.prompt(q, kv, kv, None, [m], [1], True, 0.125)
    assert ref.close(out, want, tol) <= 1 and ref.close(lse, wl, ltol) <= 1


@pytest.mark.parametrize("fmt", ["16bit", "mxfp8", "mxfp4"])
@pytest.mark.parametrize("H,N,L,R", [
    (5, 1, 512, 64), (12, 1, 512, 64), (29, 1, 512, 64), (128, 64, 512, 64),
    (5, 1, 256, 0), (12, 1, 256, 0), (29, 1, 256, 0), (128, 64, 256, 0),
    (5, 1, 480, 56), (12, 1, 480, 56), (29, 1, 288, 8)])
def test_largest_scores_that_rise_within_a_range(hip, fmt, H, N, L, R):
    """16, 32, 64 and 128 rows a block: a sequence of 40000 positions, several tiles a range, whose
    1024 different rows come again and again, with scores that rise or fall by hundreds over
    them, each row's with a slope and a sign of its own."""
    k3x, ctx = hip
    m, n = 1024, 40000
    two = N == 1  # a window of two tokens, else single ones beside the long sequence
    mla.say(f"rising scores H={H} N={N} {L}+{R} {fmt}")
    lens = [m] + [1 + 5 * i % 33 for i in range(1, N)]
    c = ref.make_cache(lens, L, R, 16, fmt, seed=H)
    g = ref.gen(H + L)
    latent = torch.randn((m, L), generator=g)
    pos = torch.arange(m)
    latent[:, 0] = torch.linspace(-30, 30, m)
    latent[:, 1] = -torch.linspace(-20, 20, m).abs()
    latent[:, 2] = torch.where(pos // 32 % 2 == 1, 16.0, -16.0)
    rotary = torch.randn((m, R), generator=g).to(BF16)
    data, values = ref.encode(latent.to(BF16), rotary, fmt)
    c["pool"][c["table"][0][pos // 16].long(), pos % 16] = data
    again = torch.arange(n) % m
    c["rows"][0] = (values[again], rotary.double()[again])
    table = torch.full((N, n // 16), -1, dtype=torch.int32)
    table[:, :m // 16] = c["table"]
    table[0] = c["table"][0].repeat(-(-n // m))[:n // 16]
    c["table"], c["lens"] = table, [n] + lens[1:]
    counts = [2] if two else [1] * N
    q = torch.randn((sum(counts), H, L + R), generator=g) * 0.1
    q[..., :3] = torch.randn((sum(counts), H, 3), generator=g) * 8
    q = q.to(BF16)
    st, out, lse = attend(hip, mla.to_device(c), q, c["lens"], 1.0, counts[0],
                          mla.offsets_of(counts))
    assert st == 0
    want, wl, tol, ltol = ref.attention(c, q, counts, 1.0)
    assert ref.close(out, want, tol) <= 1 and ref.close(lse, wl, ltol) <= 1


def test_store_past_32_bit_offsets(hip):
    """Rows 2^31 elements apart, to pages on both sides of 4 GiB."""
    k3x, ctx = hip
    L, R, page = 512, 64, 64
    pages = (5 << 30) // (page * 1152)
    pool = torch.zeros((pages, page, 1152), dtype=torch.uint8, device=DEV)
    table = mla.ints([[3, pages - 1], [pages - 2, 0]])
    wide = torch.empty((3, (1 << 31) + 64), dtype=BF16, device=DEV)
    rows = torch.randn((3, L + R), generator=ref.gen(2)).to(BF16)
    wide[:, :L + R] = rows.to(DEV)
    c = dict(pool=pool, table=table, L=L, R=R, fmt="16bit", dtype=BF16)
    mla.say("store to a pool of 5 GiB")
    assert k3x.mla_store(ctx, mla.params(k3x, c, 3), wide[:, :L], pool, table, mla.ints([65, 2]),
                         rotary=wide[:, L:L + R], offsets=mla.ints([0, 2, 3])) == 0
    assert ctx.synchronize() == 0
    data = ref.encode(rows[:, :L], rows[:, L:], "16bit")[0]
    for i, (pg, at) in enumerate([(3, 63), (pages - 1, 0), (pages - 2, 1)]):
        assert torch.equal(pool[pg, at].cpu(), data[i])
        pool[pg, at] = 0
    assert not pool.any()


def test_prompt_past_32_bit_offsets(hip):
    """Rows of queries, outputs, keys, values and rotary parts far apart: 10 GiB between the first
    key and the last."""
    k3x, ctx = hip
    m, n, H, Dn, R, Dv = 3, 40, 2, 128, 64, 128
    g = ref.gen(6)
    q = torch.randn((m, H, Dn + R), generator=g).to(BF16)
    kv = torch.randn((n, H, Dn + Dv), generator=g).to(BF16)
    rotary = torch.randn((n, R), generator=g).to(BF16)
    keys = torch.empty((n, 1 << 27), dtype=BF16, device=DEV)
    kd = keys[:, :H * (Dn + Dv)].view(n, H, Dn + Dv)
    kd.copy_(kv.to(DEV))
    rd = keys[:, 1 << 20:(1 << 20) + R]
    rd.copy_(rotary.to(DEV))
    rows = torch.empty((m, (1 << 31) + 64), dtype=BF16, device=DEV)
    qd = rows[:, :H * (Dn + R)].view(m, H, Dn + R)
    qd.copy_(q.to(DEV))
    out = rows[:, 1 << 16:(1 << 16) + H * Dv].view(m, H, Dv)
    p = k3x.make_mla_prompt_params(qd, kd[..., :Dn], kd[..., Dn:], 1, rotary=rd, scale=0.0722)
    lse = torch.zeros((m, H), device=DEV)
    mla.say("prompt over keys 2^27 elements apart")
    assert k3x.mla_prompt(ctx, p, qd, kd[..., :Dn], kd[..., Dn:], out, rotary=rd, lse=lse) == 0
    assert ctx.synchronize() == 0
    want, wl, tol, ltol = ref.prompt(q, kv[..., :Dn], kv[..., Dn:], rotary, [m], [n], True,
                                     float(torch.tensor(0.0722)))
    assert ref.close(out, want, tol) <= 1 and ref.close(lse, wl, ltol) <= 1
