"""Limits of the latent attention entry points that depend on several parameters together, checked
before the context or any device pointer is used."""
from __future__ import annotations

import ctypes as C

import pytest

pytest.importorskip("torch")
import k3x_amd as k3x  # noqa: E402
import test_mla_checks as checks  # noqa: E402

BAD = checks.BAD


@pytest.fixture(scope="module")
def lib():
    return k3x.load()


@pytest.mark.parametrize("kw", [dict(), dict(tokens=0), dict(tokens=0, sequences=65535),
                                dict(longest=1), dict(heads=1024, tokens=1 << 20),
                                dict(latent=32, rotary=0, cache_format=2)], ids=str)
def test_attention_always_takes_a_workspace(lib, kw):
    need = k3x.mla_attention_workspace_bytes(k3x.MlaParams(**{**checks.MLA, **kw}))
    assert need > 0
    for more in (dict(workspace=None), dict(bytes=need - 1), dict(bytes=0),
                 dict(workspace=(1 << 40) + 128)):
        assert checks.run(lib.k3x_hip_mla_attention, checks.ATTENTION, {**kw, **more}) == BAD


@pytest.mark.parametrize("kw", [dict(tokens=1 << 22, heads=512),
                                dict(tokens=8, longest=1 << 22, heads=512),
                                dict(tokens=1 << 22, heads=1024)], ids=str)
def test_attention_refuses_rows_past_31_bits(lib, kw):
    """Of the longest sequence; without `longest` that may have all tokens."""
    p = k3x.MlaParams(**{**checks.MLA, **kw})
    assert k3x.mla_attention_workspace_bytes(p) == 0
    assert checks.run(lib.k3x_hip_mla_attention, checks.ATTENTION, kw) == BAD
    assert k3x.mla_attention_workspace_bytes(
        k3x.MlaParams(**{**checks.MLA, **kw, "longest": 1 << 20})) > 0


@pytest.mark.parametrize("kw", [dict(tokens=1 << 22, heads=512), dict(tokens=1 << 21, heads=1024),
                                dict(tokens=65535, sequences=65535, heads=256)], ids=str)
def test_prompt_refuses_launches_past_32_bits(lib, kw):
    """Blocks of 128 queries (of every sequence one that is not full) times heads, of 256 threads."""
    assert checks.prompt(lib, **kw) == BAD


@pytest.mark.parametrize("name", ["k_stride", "v_stride", "rotary_stride"])
def test_prompt_refuses_keys_too_far_apart(lib, name):
    assert checks.prompt(lib, **{name: (1 << 27) + 8}) == BAD


def test_prompt_refuses_heads_that_make_rows_too_long(lib):
    assert checks.prompt(lib, heads=64, k_head_stride=1 << 22) == BAD
    assert checks.prompt(lib, heads=64, v_head_stride=1 << 22) == BAD
