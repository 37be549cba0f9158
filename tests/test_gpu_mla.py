"""Latent attention over a paged cache (k3x_hip_mla_store, _load and _attention) against a plain
implementation in 64 bits, at the sizes, pages and lengths where it can go wrong.  Written rows
are compared byte by byte, read ones by value, attention within the tolerance that
mla_reference.softmax_rows derives."""
from __future__ import annotations

import math

import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")
import mla_reference as ref  # noqa: E402

DEV = "cuda:0"
BF16, F16 = torch.bfloat16, torch.float16
FORMATS = [("16bit", BF16), ("16bit", F16), ("mxfp8", BF16), ("mxfp4", BF16)]
IDS = ["bf16", "fp16", "mxfp8", "mxfp4"]


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


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def offsets_of(counts):
    return ints([sum(counts[:i]) for i in range(len(counts) + 1)])


def params(k3x, cache, T, H=1, scale=1.0, eps=0.0, longest=0):
    fmt = {"16bit": k3x.CACHE_16BIT, "mxfp8": k3x.CACHE_MXFP8, "mxfp4": k3x.CACHE_MXFP4}
    return k3x.make_mla_params(cache["pool"], cache["table"], T, cache["L"], cache["R"], H,
                               fmt[cache["fmt"]], cache["dtype"], scale, eps, longest)


def to_device(cache):
    return dict(cache, pool=cache["pool"].to(DEV), table=cache["table"].to(DEV))


# ---- store and load ------------------------------------------------------------------------------

def store_case(hip, counts, lens, L, R, page, fmt, dtype, norm=True, seed=0, scale=1.0, odd=0,
               eps=1e-6):
    """Stores into a cache that holds other rows, compares every byte of the pool, loads back."""
    k3x, ctx = hip
    say(f"store {counts} of {lens} L={L} R={R} page={page} {fmt} {dtype} norm={norm} odd={odd}")
    cache = ref.make_cache(lens, L, R, page, fmt, dtype, seed)
    g = ref.gen(seed + 1)
    T = sum(counts)
    wide = torch.randn((T, L + R + odd), generator=g) * scale
    wide = wide.to(dtype).to(DEV)
    latent, rotary = wide[:, :L], wide[:, L:L + R]
    gamma = (1 + 0.3 * torch.randn(L, generator=g)).to(DEV) if norm else None
    d = to_device(cache)
    p = params(k3x, d, T, eps=eps)
    assert k3x.mla_row_bytes(L, R, p.cache_format) == cache["pool"].shape[2]
    st = k3x.mla_store(ctx, p, latent, d["pool"], d["table"], ints(lens),
                       rotary=rotary if R else None, offsets=offsets_of(counts), gamma=gamma)
    assert (st, ctx.synchronize()) == (0, 0)
    x = latent.cpu()
    if norm:
        y = x.double()
        y = y / torch.sqrt((y * y).mean(-1, keepdim=True) + float(torch.tensor(eps)))
        x = (y * gamma.cpu().double()).float().to(dtype)
    data, values = ref.encode(x, rotary.cpu(), fmt)
    want = cache["pool"].clone()
    first, kept = 0, []
    for n, m in enumerate(counts):
        for i in range(m):
            pos = lens[n] - m + i
            if pos >= 0:
                want[cache["table"][n, pos // page], pos % page] = data[first + i]
                kept.append(first + i)
        first += m
    assert torch.equal(d["pool"].cpu(), want)
    back = torch.full((T + 1, L), 7.0, dtype=dtype, device=DEV)
    turned = torch.full((T + 1, R), 7.0, dtype=dtype, device=DEV) if R else None
    st = k3x.mla_load(ctx, params(k3x, d, T + 1), d["pool"], d["table"], ints(lens), back,
                      rotary=turned, offsets=offsets_of(counts))
    assert (st, ctx.synchronize()) == (0, 0)
    hold = torch.full((T + 1, L), 7.0, dtype=torch.float64)
    hold[kept] = values[kept]
    assert torch.equal(back.cpu().double(), hold)
    if R:
        hold = torch.full((T + 1, R), 7.0, dtype=torch.float64)
        hold[kept] = rotary.cpu().double()[kept]
        assert torch.equal(turned.cpu().double(), hold)


@pytest.mark.parametrize("fmt,dtype", FORMATS, ids=IDS)
@pytest.mark.parametrize("counts,lens,page", [
    ([1], [1], 64), ([1] * 5, [7, 1, 64, 65, 129], 64), ([3, 0, 5, 1], [3, 9, 70, 33], 16),
    ([40, 1, 23], [40, 100, 25], 7), ([2, 3, 1], [0, 1, 1], 4), ([200], [333], 1),
    ([1] * 70 + [0] * 70 + [2] * 3, [5] * 143, 3)], ids=str)
@pytest.mark.parametrize("L,R", [(512, 64), (64, 0), (160, 40)])
def test_store_and_load(hip, fmt, dtype, counts, lens, page, L, R):
    store_case(hip, counts, lens, L, R, page, fmt, dtype)


@pytest.mark.parametrize("fmt,dtype", FORMATS, ids=IDS)
@pytest.mark.parametrize("L,R", [(32, 8), (96, 16), (288, 56), (480, 24), (512, 0)])
@pytest.mark.parametrize("odd", [0, 1, 4])
def test_store_widths_and_strides(hip, fmt, dtype, L, R, odd):
    store_case(hip, [9, 4], [9, 20], L, R, 8, fmt, dtype, norm=odd != 4, odd=odd)


@pytest.mark.parametrize("fmt,dtype", FORMATS, ids=IDS)
@pytest.mark.parametrize("scale", [1e-38, 1e-30, 3e-5, 2e4, 1e30], ids=str)
def test_store_of_every_size(hip, fmt, dtype, scale):
    """Scales from the least to the largest; without the norm, so that values go as they are."""
    if dtype == F16 and not 1e-6 < scale < 1e4:
        scale = 6e-8 if scale < 1 else 1e4
    store_case(hip, [17], [40], 128, 16, 16, fmt, dtype, norm=False, scale=scale)


@pytest.mark.parametrize("fmt", ["mxfp8", "mxfp4"])
def test_every_code_and_border(hip, fmt):
    """Every bf16 number of a few binades around the codes, their half-way points among them."""
    k3x, ctx = hip
    top = 448.0 if fmt == "mxfp8" else 6.0
    low = torch.arange(0, 0x4400, dtype=torch.int32).to(torch.int16).view(BF16)  # 0 .. 512
    x = low[(low <= top) & (low >= 2.0 ** -12)]
    x = torch.cat([x, x.new_zeros((-len(x)) % 31)]).view(-1, 31)
    x = torch.cat([x, torch.full((len(x), 1), top, dtype=BF16)], 1)  # the scale is 1
    x = torch.cat([x, -x], 1).contiguous()
    T = x.shape[0]
    cache = to_device(ref.make_cache([T], 64, 0, 32, fmt))
    p = params(k3x, cache, T)
    back = torch.zeros((T, 64), dtype=BF16, device=DEV)
    xd = x.to(DEV)
    say(f"every code of {fmt}")
    assert k3x.mla_store(ctx, p, xd, cache["pool"], cache["table"], ints([T])) == 0
    assert k3x.mla_load(ctx, p, cache["pool"], cache["table"], ints([T]), back) == 0
    assert ctx.synchronize() == 0
    _, _, values = ref.quantise(x, fmt)
    assert torch.equal(back.cpu().double(), values)


@pytest.mark.parametrize("fmt,dtype", FORMATS, ids=IDS)
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf], ids=str)
def test_store_latches_values_that_are_not_finite(hip, fmt, dtype, bad):
    k3x, ctx = hip
    for part in ("latent", "rotary"):
        cache = ref.make_cache([4], 64, 8, 4, fmt, dtype)
        d = to_device(cache)
        x = torch.ones((4, 72), dtype=dtype, device=DEV)
        x[2, 63 if part == "latent" else 71] = bad
        say(f"store of {bad} in {part}, {fmt}")
        assert k3x.mla_store(ctx, params(k3x, d, 4), x[:, :64], d["pool"], d["table"], ints([4]),
                             rotary=x[:, 64:]) == 0
        assert ctx.synchronize() == k3x.ERR_INVALID_MXFP4
        row = cache["table"][0, 0]
        assert torch.equal(d["pool"].cpu()[row, 2], cache["pool"][row, 2])  # as it was
        assert ctx.synchronize() == 0


# ---- attention -----------------------------------------------------------------------------------

def attend_case(hip, counts, lens, H, L=512, R=64, page=64, fmt="16bit", dtype=BF16, seed=0,
                scale=None, offsets=True, extra=0, longest=True, spread=1.0, **kw):
    k3x, ctx = hip
    say(f"attention {counts} of {lens} H={H} L={L} R={R} page={page} {fmt} {dtype} "
        f"extra={extra} {kw}")
    scale = (128 + R) ** -0.5 if scale is None else scale
    scale = float(torch.tensor(scale))
    cache = ref.make_cache(lens, L, R, page, fmt, dtype, seed, **kw)
    T = sum(counts)
    q = (torch.randn((T + extra, H, L + R), generator=ref.gen(seed + 5)) * spread).to(dtype)
    d = to_device(cache)
    qd = q.to(DEV)
    out = torch.full((T + extra, H, L), 7.0, dtype=dtype, device=DEV)
    lse = torch.full((T + extra, H), 7.0, device=DEV)
    p = params(k3x, d, T + extra, H, scale, longest=max(counts) if longest else 0)
    n = k3x.mla_attention_workspace_bytes(p)
    ws = torch.full((n,), 255, dtype=torch.uint8, device=DEV) if n else None
    st = k3x.mla_attention(ctx, p, qd, d["pool"], d["table"], ints(lens), out,
                           offsets=offsets_of(counts) if offsets else None, lse=lse, workspace=ws)
    assert (st, ctx.synchronize()) == (0, 0)
    want, wl, tol, ltol = ref.attention(cache, q, counts, scale)
    assert (out[T:] == 7).all() and (lse[T:] == 7).all()
    a, b = ref.close(out[:T], want, tol), ref.close(lse[:T], wl, ltol)
    assert a <= 1 and b <= 1, (a, b)
    return out, lse


@pytest.mark.parametrize("fmt,dtype", FORMATS, ids=IDS)
@pytest.mark.parametrize("H", [1, 16, 20, 64, 128])
@pytest.mark.parametrize("lens", [[1], [31, 32, 33], [64, 0, 97, 128, 1, 300]], ids=str)
def test_decode(hip, fmt, dtype, H, lens):
    attend_case(hip, [1] * len(lens), lens, H, fmt=fmt, dtype=dtype)


@pytest.mark.parametrize("fmt,dtype", FORMATS, ids=IDS)
@pytest.mark.parametrize("counts,lens,H", [
    ([5, 5, 5], [40, 5, 97], 8), ([3, 0, 8, 1], [33, 50, 8, 65], 32), ([2, 5], [1, 3], 40),
    ([9], [200], 16), ([40], [40], 8), ([4, 4], [0, 70], 3)], ids=str)
def test_windows(hip, fmt, dtype, counts, lens, H):
    """Drafted tokens see themselves and what is before them; tokens at positions below 0 none."""
    attend_case(hip, counts, lens, H, fmt=fmt, dtype=dtype)


@pytest.mark.parametrize("page", [1, 2, 7, 16, 33, 128, 1000])
@pytest.mark.parametrize("fmt", ["16bit", "mxfp8", "mxfp4"])
def test_pages(hip, page, fmt):
    attend_case(hip, [1, 2, 1], [50, 129, 200], 16, page=page, fmt=fmt)


@pytest.mark.parametrize("L,R", [(32, 0), (64, 16), (96, 8), (160, 40), (256, 64), (256, 0),
                                 (384, 64), (480, 56), (512, 0), (512, 32)])
@pytest.mark.parametrize("fmt,dtype", FORMATS, ids=IDS)
def test_widths(hip, L, R, fmt, dtype):
    attend_case(hip, [1, 3], [70, 45], 24, L, R, 16, fmt, dtype)


@pytest.mark.parametrize("fmt", ["16bit", "mxfp8", "mxfp4"])
def test_long(hip, fmt):
    attend_case(hip, [1], [5003], 16, fmt=fmt)
    attend_case(hip, [1, 2], [2600, 1111], 64, fmt=fmt)
    attend_case(hip, [1], [3500], 128, fmt=fmt)


@pytest.mark.parametrize("N", [65, 300])
def test_many_sequences(hip, N):
    lens = [1 + 7 * n % 90 for n in range(N)]
    attend_case(hip, [1] * N, lens, 4, 64, 16, 16)
    counts = [n % 3 for n in range(N)]
    attend_case(hip, counts, [max(a, b) for a, b in zip(lens, counts)], 4, 64, 16, 16, extra=3)


@pytest.mark.parametrize("fmt,dtype", FORMATS, ids=IDS)
@pytest.mark.parametrize("L,R", [(512, 64), (256, 0), (160, 8)])
def test_many_sequences_of_many_rows(hip, fmt, dtype, L, R):
    """Enough rows for the largest blocks, part of them empty, one sequence in many ranges."""
    lens = [900, 0, 1, 33] + [1 + 11 * n % 70 for n in range(61)]
    attend_case(hip, [1] * 65, lens, 68, L, R, 16, fmt, dtype)
    counts = [n % 3 for n in range(33)]
    lens = [max(a, b) for a, b in zip(lens, counts)]
    attend_case(hip, counts, lens, 100, L, R, 64, fmt, dtype, extra=2, spread=4.0)


@pytest.mark.parametrize("fmt,dtype", FORMATS, ids=IDS)
@pytest.mark.parametrize("L,R", [(512, 64), (96, 8)])
def test_more_row_blocks_than_a_group(hip, fmt, dtype, L, R):
    """Long windows beside single tokens: groups of row blocks, several a range and cut between
    ranges, with and without `longest`."""
    attend_case(hip, [270, 0, 31], [300, 50, 20], 128, L, R, 16, fmt, dtype, extra=3)
    attend_case(hip, [1, 70] + [1, 2] * 3, [900, 400, 5, 2, 300, 3, 1, 64], 24, L, R, 16, fmt, dtype,
                longest=False)
    k3x, _ = hip
    p = params(k3x, to_device(ref.make_cache([9], L, R, 16, fmt, dtype)), 1 << 14, 128)
    assert k3x.mla_attention_workspace_bytes(p) <= 1 << 28


def test_without_offsets(hip):
    attend_case(hip, [2, 2, 2], [30, 2, 64], 16, offsets=False, longest=False)
    attend_case(hip, [3], [64], 16, offsets=True, longest=False, extra=2)


def test_sharp_scores(hip):
    """One key takes nearly all; the running largest score rises late."""
    attend_case(hip, [1, 1], [600, 90], 16, spread=12.0)
    attend_case(hip, [1, 1], [600, 90], 64, scale=1e-3)


def test_rising_scores(hip):
    """Every tile's scores pass the last one's by far, then fall far below."""
    k3x, ctx = hip
    n, L = 320, 64
    cache = ref.make_cache([n], L, 0, 16, junk=False)
    ramp = torch.linspace(-40, 40, n).abs().neg() * 30
    rows = torch.randn((n, L), generator=ref.gen(1))
    rows[:, 0] = ramp
    latent = rows.to(BF16)
    data, values = ref.encode(latent, torch.zeros((n, 0), dtype=BF16), "16bit")
    pos = torch.arange(n)
    cache["pool"][cache["table"][0][pos // 16].long(), pos % 16] = data
    cache["rows"] = [(values, torch.zeros((n, 0), dtype=torch.float64))]
    for sign in (1.0, -1.0):
        q = torch.zeros((1, 3, L), dtype=BF16)
        q[:, :, 0], q[:, 1, 1] = sign, 0.5
        d = to_device(cache)
        out = torch.zeros((1, 3, L), dtype=BF16, device=DEV)
        lse = torch.zeros((1, 3), device=DEV)
        p = params(k3x, d, 1, 3)
        m = k3x.mla_attention_workspace_bytes(p)
        ws = torch.empty((m,), dtype=torch.uint8, device=DEV) if m else None
        say(f"rising scores {sign}")
        assert k3x.mla_attention(ctx, p, q.to(DEV), d["pool"], d["table"], ints([n]), out,
                                 lse=lse, workspace=ws) == 0
        assert ctx.synchronize() == 0
        want, wl, tol, ltol = ref.attention(cache, q, [1], 1.0)
        assert ref.close(out, want, tol) <= 1 and ref.close(lse, wl, ltol) <= 1


def test_attention_latches_rows_that_are_not_finite(hip):
    k3x, ctx = hip
    for where in ("q", "latent", "rotary"):
        cache = ref.make_cache([40, 40], 64, 16, 8)
        d = to_device(cache)
        q = torch.ones((2, 4, 80), dtype=BF16, device=DEV)
        if where == "q":
            q[1, 2, 3] = math.nan
        else:
            row = cache["table"][1, 2].long()
            d["pool"][row, 5].view(BF16)[3 if where == "latent" else 70] = math.inf
        p = params(k3x, d, 2, 4)
        n = k3x.mla_attention_workspace_bytes(p)
        ws = torch.empty((n,), dtype=torch.uint8, device=DEV) if n else None
        out = torch.zeros((2, 4, 64), dtype=BF16, device=DEV)
        say(f"attention with infinity in {where}")
        assert k3x.mla_attention(ctx, p, q, d["pool"], d["table"], ints([40, 40]), out,
                                 workspace=ws) == 0
        assert ctx.synchronize() == k3x.ERR_INVALID_MXFP4
        assert ctx.synchronize() == 0


@pytest.mark.parametrize("what", ["offsets fall", "offsets past", "length", "page", "longest"])
def test_unfit_sequences_are_latched(hip, what):
    k3x, ctx = hip
    cache = ref.make_cache([40, 40], 64, 16, 8)
    d = to_device(cache)
    lens, offs = ints([40, 40]), ints([0, 1, 2])
    longest = 0
    if what == "offsets fall":
        offs = ints([0, 2, 1])
    elif what == "offsets past":
        offs = ints([0, 1, 3])
    elif what == "length":
        lens = ints([40, 41])
    elif what == "page":
        d["table"][1, 4] = cache["pool"].shape[0]
    else:
        offs, longest = ints([0, 0, 2]), 1
    x = torch.ones((2, 4, 80), dtype=BF16, device=DEV)
    guard = torch.full((4, 4, 64), 7.0, dtype=BF16, device=DEV)
    out = guard[1:3]
    p = params(k3x, d, 2, 4, longest=longest)
    n = k3x.mla_attention_workspace_bytes(p)
    ws = torch.empty((n,), dtype=torch.uint8, device=DEV) if n else None
    calls = [
        lambda: k3x.mla_attention(ctx, p, x, d["pool"], d["table"], lens, out, offsets=offs,
                                  workspace=ws),
        lambda: k3x.mla_store(ctx, p, x[:, 0, :64], d["pool"], d["table"], lens,
                              rotary=x[:, 0, 64:], offsets=offs),
        lambda: k3x.mla_load(ctx, p, d["pool"], d["table"], lens, out[:, 0], offsets=offs)]
    for i, call in enumerate(calls):
        if what == "page" and i:  # the last position's page only
            d["table"][1, 4] = -1
        say(f"{what}, call {i}")
        assert call() == 0
        assert ctx.synchronize() == k3x.ERR_INVALID_STATE
        assert (guard[0] == 7).all() and (guard[3] == 7).all()
    assert ctx.synchronize() == 0


def test_past_32_bit_offsets(hip):
    """Pages on both sides of 4 GiB, rows of q and out far apart."""
    k3x, ctx = hip
    L, R, page = 512, 64, 64
    small = ref.make_cache([150, 70], L, R, page, seed=3, junk=False)
    pages = (5 << 30) // (page * 1152)
    pool = torch.empty((pages, page, 1152), dtype=torch.uint8, device=DEV)
    # The small pool's pages, spread from the first to the last of the large one.
    to = torch.linspace(0, pages - 1, small["pool"].shape[0]).long()
    pool[to.to(DEV)] = small["pool"].to(DEV)
    table = to[small["table"].long()].int().to(DEV)
    d = dict(small, pool=pool, table=table)
    wide = torch.zeros((2, (1 << 31) + 64), dtype=BF16, device=DEV)
    q = torch.randn((2, 16, L + R), generator=ref.gen(9)).to(BF16)
    qd = wide[:, :16 * (L + R)].view(2, 16, L + R)
    qd.copy_(q.to(DEV))
    out = torch.zeros((2, 16, L), dtype=BF16, device=DEV)
    lse = torch.zeros((2, 16), device=DEV)
    p = params(k3x, d, 2, 16, 0.0722, longest=1)
    n = k3x.mla_attention_workspace_bytes(p)
    ws = torch.empty((n,), dtype=torch.uint8, device=DEV) if n else None
    say("pool of 5 GiB")
    assert k3x.mla_attention(ctx, p, qd, pool, table, ints([150, 70]), out, lse=lse,
                             workspace=ws) == 0
    assert ctx.synchronize() == 0
    want, wl, tol, ltol = ref.attention(small, q, [1, 1], float(torch.tensor(0.0722)))
    assert ref.close(out, want, tol) <= 1 and ref.close(lse, wl, ltol) <= 1
    back = torch.zeros((220, L), dtype=BF16, device=DEV)
    assert k3x.mla_load(ctx, params(k3x, d, 220), pool, table, ints([150, 70]), back,
                        offsets=ints([0, 150, 220])) == 0
    assert ctx.synchronize() == 0
    assert torch.equal(back.cpu().double(), torch.cat([r[0] for r in small["rows"]]))
