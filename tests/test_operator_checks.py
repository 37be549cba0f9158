"""Refusals of the routing, delta rule and verification entry points: checked
before the context or any device pointer is used, so a zeroed buffer stands in
for both and no GPU is needed."""
from __future__ import annotations

import ctypes as C
import math
import os
import re
from decimal import Decimal, localcontext
from fractions import Fraction

import pytest

torch = pytest.importorskip("torch")
import k3x_amd as k3x  # noqa: E402

CTX = C.create_string_buffer(1 << 16)
P = 1 << 20  # a pointer that is never followed
BAD = k3x.ERR_INVALID_EXTENT


@pytest.fixture(scope="module")
def lib():
    return k3x.load()


def ctx():
    return C.cast(CTX, C.c_void_p)


ROUTE = dict(tokens=4, experts=64, top_k=8, dtype=0, scoring=0, renorm=0, routed_scale=1.0,
             groups=8, top_groups=4, group_score=0, logits_stride=0)


def route(lib, logits=P, bias=None, ids=P, weights=P, c=None, **kw):
    p = k3x.RouteParams(**dict(ROUTE, **kw))
    return lib.k3x_hip_route(ctx() if c is None else c, C.byref(p), logits, bias, ids, weights)


@pytest.mark.parametrize("kw", [
    dict(tokens=0), dict(tokens=(1 << 20) + 1), dict(experts=0), dict(experts=4104), dict(top_k=0),
    dict(top_k=33), dict(top_k=65, experts=4096), dict(dtype=2), dict(scoring=2), dict(renorm=3),
    dict(routed_scale=math.nan), dict(routed_scale=math.inf), dict(groups=0), dict(groups=7),
    dict(groups=128, experts=256), dict(top_groups=0), dict(top_groups=9), dict(group_score=2),
    dict(logits_stride=63), dict(logits=None), dict(ids=None), dict(weights=None),
    dict(logits=P + 2), dict(bias=P + 1), dict(ids=P + 2), dict(weights=P + 3),
    dict(logits=P + 1, dtype=1)], ids=str)
def test_route_refuses(lib, kw):
    assert route(lib, **kw) == BAD


def test_null_contexts(lib):
    assert lib.k3x_hip_route(None, None, None, None, None, None) == BAD
    assert lib.k3x_hip_route(ctx(), None, P, None, P, P) == BAD
    assert lib.k3x_hip_delta_rule(None, None, *[None] * 12, 0) == BAD
    assert lib.k3x_hip_verify_draft(None, None, *[None] * 9, 0) == BAD
    assert lib.k3x_hip_delta_workspace(None) == 0
    assert lib.k3x_hip_verify_workspace(None) == 0


DELTA = dict(sequences=2, tokens=200, key_heads=2, value_heads=4, key_dim=128, value_dim=128,
             dtype=1, gate=2, scale=1.0, norm_epsilon=1e-6, longest=0, slots=2, q_stride=0,
             k_stride=0, v_stride=0, out_stride=0)
DELTA_PTRS = dict(q=P, k=P, v=P, g=P, beta=P, offsets=P, limits=None, slot_index=None,
                  state_in=1 << 30, state_out=1 << 32, out=P, workspace=1 << 40, bytes=1 << 40)


def delta(lib, **kw):
    p = k3x.DeltaParams(**{**DELTA, **{x: y for x, y in kw.items() if x in DELTA}})
    a = {**DELTA_PTRS, **{x: y for x, y in kw.items() if x not in DELTA}}
    return lib.k3x_hip_delta_rule(ctx(), C.byref(p), *a.values())


@pytest.mark.parametrize("kw", [
    dict(sequences=0), dict(sequences=65536), dict(tokens=(1 << 24) + 1), dict(key_heads=0),
    dict(key_heads=3), dict(value_heads=0), dict(value_heads=1026), dict(key_dim=0),
    dict(key_dim=257), dict(value_dim=0), dict(value_dim=1025), dict(dtype=3), dict(gate=3),
    dict(gate=0), dict(g=None), dict(scale=math.inf), dict(norm_epsilon=-1e-6),
    dict(norm_epsilon=math.nan), dict(slots=0), dict(slots=1), dict(q_stride=255),
    dict(k_stride=1), dict(v_stride=511), dict(out_stride=3), dict(q_stride=1 << 32),
    dict(offsets=None, tokens=201), dict(q=None), dict(k=None), dict(v=None), dict(beta=None),
    dict(out=None), dict(q=P + 1), dict(out=P + 1), dict(dtype=0, v=P + 2), dict(g=P + 2),
    dict(beta=P + 1), dict(offsets=P + 2), dict(limits=P + 1), dict(slot_index=P + 3),
    dict(state_in=P + 8), dict(state_out=P + 4),
    dict(state_out=(1 << 30) + 16), dict(state_out=(1 << 30) - 2 * 4 * 128 * 128 * 4 + 16)],
    ids=str)
def test_delta_refuses(lib, kw):
    assert delta(lib, **kw) == BAD


def test_delta_workspace(lib):
    """A call that needs a workspace refuses one that is missing, short or off alignment."""
    p = k3x.DeltaParams(**dict(DELTA, tokens=4096, longest=2048))
    need = k3x.delta_workspace_bytes(p)
    assert lib.k3x_hip_delta_workspace(C.byref(k3x.DeltaParams(**dict(DELTA, key_dim=0)))) == 0
    assert lib.k3x_hip_delta_workspace(C.byref(k3x.DeltaParams(**dict(DELTA, tokens=2)))) == 0
    if need:
        big = dict(tokens=4096, longest=2048)
        assert delta(lib, workspace=None, **big) == BAD
        assert delta(lib, bytes=need - 1, **big) == BAD
        assert delta(lib, workspace=(1 << 40) + 128, **big) == BAD


VERIFY = dict(sequences=2, drafts=4, vocab=1000, dtype=0, form=0, greedy=0, temperature=1.0,
              row_stride=0)
VERIFY_PTRS = dict(target=P, draft=P, tokens=P, draft_counts=None, accept_u=P, sample_u=P,
                   accepted=P, out_tokens=P, workspace=P, bytes=1 << 40)


def verify(lib, **kw):
    p = k3x.VerifyParams(**{**VERIFY, **{x: y for x, y in kw.items() if x in VERIFY}})
    a = {**VERIFY_PTRS, **{x: y for x, y in kw.items() if x not in VERIFY}}
    return lib.k3x_hip_verify_draft(ctx(), C.byref(p), *a.values())


@pytest.mark.parametrize("kw", [
    dict(sequences=0), dict(sequences=65536), dict(drafts=65), dict(vocab=0),
    dict(vocab=(1 << 20) + 1), dict(dtype=2), dict(form=2), dict(greedy=2), dict(temperature=0.0),
    dict(temperature=-1.0), dict(temperature=math.nan), dict(temperature=math.inf),
    dict(row_stride=999), dict(target=None), dict(tokens=None), dict(accept_u=None),
    dict(sample_u=None), dict(accepted=None), dict(out_tokens=None), dict(workspace=None),
    dict(bytes=255), dict(workspace=P + 128), dict(target=P + 2), dict(draft=P + 1),
    dict(tokens=P + 2), dict(draft_counts=P + 1), dict(accept_u=P + 2), dict(sample_u=P + 2),
    dict(accepted=P + 1), dict(out_tokens=P + 2)], ids=str)
def test_verify_refuses(lib, kw):
    assert verify(lib, **kw) == BAD


def test_more_threads_than_a_launch(lib):
    """Extents that are each allowed, whose product is no launch (2^32 threads)."""
    assert delta(lib, sequences=32768, value_heads=1024, slots=32768) == BAD
    assert delta(lib, sequences=1, tokens=1 << 24, value_heads=1024, longest=1 << 24) == BAD
    assert verify(lib, sequences=65535, drafts=64, vocab=1 << 20) == BAD


def test_binding_checks_tensors():
    """The binding's own checks come before any pointer is taken."""
    class Fake:
        handle, lib = None, None

    p = k3x.make_route_params(2, 8, 2)
    x = torch.zeros((2, 8))
    with pytest.raises(ValueError):
        k3x.route(Fake, p, x.double(), torch.zeros((2, 2), dtype=torch.int32), torch.zeros((2, 2)))
    with pytest.raises(ValueError):
        k3x.route(Fake, p, x, torch.zeros((2, 2), dtype=torch.int64), torch.zeros((2, 2)))
    with pytest.raises(ValueError):
        k3x.route(Fake, p, x[:1], torch.zeros((2, 2), dtype=torch.int32), torch.zeros((2, 2)))
    q = torch.zeros((3, 1, 4))
    d = k3x.make_delta_params(q, q, q, 1)
    with pytest.raises(ValueError):
        k3x.delta_rule(Fake, d, q, q.bfloat16(), q, torch.zeros((3, 1)), q)
    with pytest.raises(ValueError):
        k3x.delta_rule(Fake, d, q, q, q, torch.zeros((3, 1)), q, offsets=torch.zeros(2))
    t = torch.zeros((1, 3, 9))
    v = k3x.make_verify_params(t)
    ints = torch.zeros((1, 3), dtype=torch.int32)
    with pytest.raises(ValueError):
        k3x.verify_draft(Fake, v, t, ints, ints[0, :1], ints)


def test_strides_of_rows():
    """Rows that lie apart keep their distance; packed ones and single rows have none."""
    wide = torch.zeros((4, 30))
    assert k3x._row_stride(wide) == 0
    assert k3x._row_stride(wide[:, 3:9]) == 30
    assert k3x._row_stride(wide[:1, 3:9]) == 0
    assert k3x._row_stride(wide[:, 2:26].unflatten(1, (2, 12))) == 30
    for bad in (wide.t(), wide.unflatten(1, (2, 15))[:, :, :5]):
        with pytest.raises(ValueError):
            k3x._row_stride(bad)


class Recorded:
    """A context whose library calls are kept and not made."""
    handle, device = None, 0

    def __init__(self):
        self.lib, self.calls = self, []

    def __getattr__(self, name):
        return lambda *a: self.calls.append((name, a)) or 0


class OnDevice(torch.Tensor):
    """A tensor that says it is on device 0."""
    is_cuda = True

    def get_device(self):
        return 0


def there(x):
    return x.as_subclass(OnDevice)


def verified(target, draft=None, params=None):
    """The parameters that verify_draft calls the library with."""
    N, D1, V = target.shape
    c, ints = Recorded(), torch.zeros((N, D1), dtype=torch.int32)
    p = k3x.make_verify_params(target) if params is None else params
    u = torch.zeros((N, D1))
    assert k3x.verify_draft(c, p, there(target), there(ints[:, 1:].contiguous()),
                            there(ints[:, 0].contiguous()), there(ints),
                            draft=None if draft is None else there(draft),
                            accept_u=there(u[:, 1:].contiguous()),
                            sample_u=there(u[:, 0].contiguous())) == 0
    (name, args), = c.calls
    assert name == "k3x_hip_verify_draft"
    return args[1]._obj


def test_verified_rows_lie_where_the_tensors_say():
    """The distance of rows is the tensors' own, whatever the parameters hold: a distance set
    there would be read past the end of packed rows."""
    packed = torch.zeros((2, 4, 9))
    p = k3x.make_verify_params(packed)
    p.row_stride = 1 << 20
    assert verified(packed, packed[:, :3].contiguous(), p).row_stride in (0, 9)
    assert p.row_stride == 1 << 20  # the caller's own is left
    wide = torch.zeros((2, 4, 13))[..., :9]
    assert verified(wide).row_stride == 13
    assert verified(wide, torch.zeros((2, 3, 13))[..., :9]).row_stride == 13
    assert verified(torch.zeros((5, 1, 13))[..., 2:11]).row_stride == 13
    assert verified(torch.zeros((1, 5, 13))[..., 2:11]).row_stride == 13
    one = torch.zeros((1, 2, 13))[..., :9]  # a single drafted row lies anywhere
    assert verified(one, torch.zeros((1, 1, 30))[..., :9]).row_stride == 13
    assert verified(one, torch.zeros((1, 1, 9))).row_stride == 13


@pytest.mark.parametrize("target,draft", [
    (torch.zeros((2, 4, 13))[..., :9], torch.zeros((2, 3, 9))),
    (torch.zeros((2, 4, 9)), torch.zeros((2, 3, 13))[..., :9]),
    (torch.zeros((2, 5, 9))[:, :4], None),
    (torch.zeros((4, 2, 9)).transpose(0, 1), None),
    (torch.zeros((2, 4, 18))[..., ::2], None),
    (torch.zeros((1, 1, 9)).expand(2, 4, 9), None),
    (torch.zeros(40).as_strided((2, 4, 9), (16, 4, 1)), None),
    (torch.empty((2, 4, 9), device="meta").as_strided((2, 4, 9), (1 << 34, 1 << 32, 1)), None)],
    ids=["draft_packed", "target_packed", "gap", "transposed", "every_second", "one_row", "overlap",
         "far"])
def test_verified_rows_that_do_not_lie_evenly(target, draft):
    with pytest.raises(ValueError):
        verified(target, draft)


@pytest.mark.parametrize("far,refused", [(64, False), (80, False), ((1 << 32) - 1, False),
                                         (1 << 32, True), ((1 << 32) + 80, True)])
def test_distance_of_logits(far, refused):
    """A distance past the parameter's 32 bits is refused, not cut to them."""
    c, p = Recorded(), k3x.make_route_params(2, 64, 4)
    logits = there(torch.empty((2, 64), device="meta").as_strided((2, 64), (far, 1)))
    ids, weights = there(torch.zeros((2, 4), dtype=torch.int32)), there(torch.zeros((2, 4)))
    if refused:
        with pytest.raises(ValueError):
            k3x.route(c, p, logits, ids, weights)
        assert not c.calls
    else:
        assert k3x.route(c, p, logits, ids, weights) == 0
        assert c.calls[0][1][1]._obj.logits_stride == (0 if far == 64 else far)


def test_bound_of_the_exponential_in_verification():
    """The series of verify.hip's 2^f against 60 digits over |f| <= 1/2, exactly as its
    coefficients are held: within the bound that its comment states."""
    path = os.path.join(os.path.dirname(k3x.__file__), "csrc", "verify.hip")
    with open(path) as f:
        source = f.read()
    at = source.index("inline double exp2_f64")
    bound = float(re.findall(r"([0-9.]+e-[0-9]+) of it at most", source[:at])[-1])
    body = source[at:source.index("ldexp", at)]
    series = [Fraction(float(x or y)) for x, y in
              re.findall(r"double p = ([0-9.e+-]+);|p, f, ([0-9.e+-]+)\)", body)]
    assert len(series) == 12
    worst = 0.0
    with localcontext() as digits:
        digits.prec = 60
        for i in range(-256, 257):
            f, p = Fraction(i, 512), Fraction(0)
            for c in series:
                p = p * f + c
            want = (Decimal(2).ln() * f.numerator / f.denominator).exp()
            worst = max(worst, abs(float(Decimal(p.numerator) / p.denominator / want - 1)))
    assert worst <= bound, worst
