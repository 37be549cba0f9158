"""Refusals of the latent attention and logits entry points: checked before the context or any
device pointer is used, so a zeroed buffer stands in for both and no GPU is needed."""
from __future__ import annotations

import ctypes as C
import math

import pytest

torch = pytest.importorskip("torch")
import k3x_amd as k3x  # noqa: E402
import mla_reference as ref  # noqa: E402

CTX = C.create_string_buffer(1 << 16)
P = 1 << 20  # a pointer that is never followed
BAD = k3x.ERR_INVALID_EXTENT


@pytest.fixture(scope="module")
def lib():
    return k3x.load()


def ctx():
    return C.cast(CTX, C.c_void_p)


MLA = dict(sequences=2, tokens=4, heads=16, latent=512, rotary=64, dtype=1, cache_format=0,
           page_size=64, pages=100, table_width=10, longest=0, scale=1.0, norm_epsilon=1e-6,
           latent_stride=0, rotary_stride=0, q_stride=0, out_stride=0)
SHARED = [
    dict(sequences=0), dict(sequences=65536), dict(tokens=(1 << 22) + 1), dict(heads=0),
    dict(heads=1025), dict(latent=0), dict(latent=48), dict(latent=544), dict(rotary=72),
    dict(rotary=12), dict(dtype=0), dict(dtype=3), dict(dtype=2, cache_format=1),
    dict(dtype=2, cache_format=2), dict(cache_format=3), dict(page_size=0),
    dict(page_size=65537), dict(pages=0), dict(pages=1 << 26), dict(table_width=0),
    dict(table_width=(1 << 20) + 1), dict(scale=0.0), dict(scale=-1.0), dict(scale=math.nan),
    dict(scale=math.inf), dict(norm_epsilon=-1.0), dict(norm_epsilon=math.nan),
    dict(latent_stride=511), dict(rotary_stride=63), dict(q_stride=16 * 576 - 8),
    dict(out_stride=16 * 512 - 8), dict(latent_stride=(1 << 32) + 1), dict(table=None),
    dict(lens=None), dict(pool=None), dict(table=P + 2), dict(lens=P + 1), dict(offsets=P + 2),
    dict(pool=P + 128)]


def run(fn, ptrs, kw):
    p = k3x.MlaParams(**{**MLA, **{x: y for x, y in kw.items() if x in MLA}})
    a = {**ptrs, **{x: y for x, y in kw.items() if x not in MLA}}
    return fn(ctx(), C.byref(p), *a.values())


STORE = dict(latent_ptr=P, rotary_ptr=P, gamma=P, table=P, offsets=P, lens=P, pool=P)
LOAD = dict(pool=P, table=P, offsets=P, lens=P, latent_ptr=P, rotary_ptr=P)
ATTENTION = dict(q=P, pool=P, table=P, offsets=P, lens=P, out=P, lse=P, workspace=1 << 40,
                 bytes=1 << 50)


@pytest.mark.parametrize("kw", SHARED + [
    dict(latent_ptr=None), dict(rotary_ptr=None), dict(latent_ptr=P + 1), dict(rotary_ptr=P + 1),
    dict(gamma=P + 2)], ids=str)
def test_store_refuses(lib, kw):
    assert run(lib.k3x_hip_mla_store, STORE, kw) == BAD


@pytest.mark.parametrize("kw", SHARED + [dict(latent_ptr=None), dict(latent_ptr=P + 1),
                                         dict(rotary_ptr=P + 1)], ids=str)
def test_load_refuses(lib, kw):
    assert run(lib.k3x_hip_mla_load, LOAD, kw) == BAD


@pytest.mark.parametrize("kw", SHARED + [
    dict(q=None), dict(out=None), dict(q=P + 8), dict(out=P + 8), dict(lse=P + 2),
    dict(q_stride=16 * 576 + 4), dict(out_stride=16 * 512 + 4)], ids=str)
def test_attention_refuses(lib, kw):
    assert run(lib.k3x_hip_mla_attention, ATTENTION, kw) == BAD


def test_attention_workspace(lib):
    p = k3x.MlaParams(**MLA)
    need = k3x.mla_attention_workspace_bytes(p)
    assert lib.k3x_hip_mla_attention_workspace(None) == 0
    assert k3x.mla_attention_workspace_bytes(k3x.MlaParams(**dict(MLA, latent=40))) == 0
    if need:
        for kw in (dict(workspace=None), dict(bytes=need - 1), dict(workspace=(1 << 40) + 128)):
            assert run(lib.k3x_hip_mla_attention, ATTENTION, kw) == BAD


@pytest.mark.parametrize("fmt", ["16bit", "mxfp8", "mxfp4"])
def test_row_bytes(lib, fmt):
    code = {"16bit": 0, "mxfp8": 1, "mxfp4": 2}[fmt]
    for L in range(32, 513, 32):
        for R in range(0, 65, 8):
            n = k3x.mla_row_bytes(L, R, code)
            assert n == ref.row_bytes(L, R, fmt) and n % 16 == 0
    with pytest.raises(ValueError):
        k3x.mla_row_bytes(100, 0, code)
    assert lib.k3x_hip_mla_row_bytes(None) == 0


PROMPT = dict(sequences=2, tokens=40, keys=60, heads=4, key_dim=128, rotary=64, value_dim=128,
              dtype=1, causal=1, longest=0, scale=1.0, q_stride=0, k_stride=0, v_stride=0,
              rotary_stride=0, out_stride=0, k_head_stride=0, v_head_stride=0)
PROMPT_PTRS = dict(q=P, k=P, v=P, rotary_ptr=P, offsets=P, key_offsets=P, out=P, lse=P)


def prompt(lib, **kw):
    p = k3x.MlaPromptParams(**{**PROMPT, **{x: y for x, y in kw.items() if x in PROMPT}})
    a = {**PROMPT_PTRS, **{x: y for x, y in kw.items() if x not in PROMPT}}
    return lib.k3x_hip_mla_prompt(ctx(), C.byref(p), *a.values())


@pytest.mark.parametrize("kw", [
    dict(sequences=0), dict(sequences=65536), dict(tokens=(1 << 22) + 1),
    dict(keys=(1 << 22) + 1), dict(heads=0), dict(heads=1025), dict(key_dim=0),
    dict(key_dim=136), dict(key_dim=100), dict(rotary=72), dict(rotary=4), dict(value_dim=0),
    dict(value_dim=136), dict(value_dim=20), dict(dtype=0), dict(dtype=3), dict(causal=2),
    dict(scale=0.0), dict(scale=-2.0), dict(scale=math.nan), dict(scale=math.inf),
    dict(q_stride=4 * 192 - 8), dict(q_stride=4 * 192 + 4), dict(k_stride=120),
    dict(k_stride=4 * 128 + 4), dict(v_stride=120), dict(v_stride=513), dict(rotary_stride=56),
    dict(rotary_stride=65), dict(out_stride=4 * 128 - 8), dict(out_stride=4 * 128 + 1),
    dict(k_head_stride=120), dict(k_head_stride=129), dict(v_head_stride=120),
    dict(v_head_stride=130), dict(k_stride=1 << 33), dict(q=None), dict(k=None), dict(v=None),
    dict(rotary_ptr=None), dict(out=None), dict(q=P + 8), dict(k=P + 8), dict(v=P + 2),
    dict(rotary_ptr=P + 4), dict(out=P + 8), dict(offsets=P + 2), dict(key_offsets=P + 1),
    dict(lse=P + 2)], ids=str)
def test_prompt_refuses(lib, kw):
    assert prompt(lib, **kw) == BAD


LOGITS = dict(sequences=2, drafts=4, vocab=1000, dtype=0, row_stride=0, out_stride=0,
              history_width=10, biases=3, masks=2, mask_stride=0)
LOGITS_PTRS = dict(logits=P, history=P, history_lens=P, prompt_lens=P, draft_tokens=P,
                   draft_counts=P, repetition=P, frequency=P, presence=P, bias_offsets=P,
                   bias_tokens=P, bias_values=P, mask_rows=P, mask_index=P, out=P)


def logits(lib, **kw):
    p = k3x.LogitsParams(**{**LOGITS, **{x: y for x, y in kw.items() if x in LOGITS}})
    a = {**LOGITS_PTRS, **{x: y for x, y in kw.items() if x not in LOGITS}}
    return lib.k3x_hip_adjust_logits(ctx(), C.byref(p), *a.values())


@pytest.mark.parametrize("kw", [
    dict(sequences=0), dict(sequences=65536), dict(drafts=65), dict(vocab=0),
    dict(vocab=(1 << 20) + 1), dict(dtype=2), dict(row_stride=999), dict(out_stride=999),
    dict(mask_stride=31), dict(logits=None), dict(out=None), dict(history_lens=None),
    dict(draft_tokens=None), dict(bias_tokens=None), dict(bias_values=None),
    dict(mask_index=None)] + [
        {k: P + 2} for k in LOGITS_PTRS], ids=str)
def test_logits_refuses(lib, kw):
    assert logits(lib, **kw) == BAD


def test_null_contexts(lib):
    assert lib.k3x_hip_mla_store(None, None, *[None] * 7) == BAD
    assert lib.k3x_hip_mla_load(None, None, *[None] * 6) == BAD
    assert lib.k3x_hip_mla_attention(None, None, *[None] * 8, 0) == BAD
    assert lib.k3x_hip_mla_prompt(None, None, *[None] * 8) == BAD
    assert lib.k3x_hip_adjust_logits(None, None, *[None] * 15) == BAD


def test_binding_checks_tensors():
    """The binding's own checks come before any pointer is taken."""
    class Fake:
        handle, lib, device = None, k3x.load(), 0

    pool = torch.zeros((3, 4, k3x.mla_row_bytes(64, 8)), dtype=torch.uint8)
    table, lens = torch.zeros((2, 2), dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    p = k3x.make_mla_params(pool, table, 2, 64, 8, 4)
    x = torch.zeros((2, 64), dtype=torch.bfloat16)
    q = torch.zeros((2, 4, 72), dtype=torch.bfloat16)
    with pytest.raises(ValueError):  # on the CPU
        k3x.mla_store(Fake, p, x, pool, table, lens)
    with pytest.raises(ValueError):
        k3x.mla_store(Fake, p, x.float(), pool, table, lens)
    with pytest.raises(ValueError):
        k3x.mla_load(Fake, p, pool, table, lens, x[:, :32])
    with pytest.raises(ValueError):
        k3x.mla_attention(Fake, p, q[..., 1:], pool, table, lens, q[..., :64].contiguous())
    k = torch.zeros((5, 4, 64), dtype=torch.bfloat16)
    pp = k3x.make_mla_prompt_params(q[..., :64].contiguous(), k, k, 1)
    with pytest.raises(ValueError):
        k3x.mla_prompt(Fake, pp, q[..., :64].contiguous(), k, k.half(), q)
    l = torch.zeros((2, 3, 100))
    lp = k3x.make_logits_params(l)
    with pytest.raises(ValueError):
        k3x.adjust_logits(Fake, lp, l, l.bfloat16())
    with pytest.raises(ValueError):
        k3x.adjust_logits(Fake, lp, l.double(), l)
