"""The cache's C entry points reject invalid arguments with the documented codes before any CUDA
call, and the oracle's layout is a bijection.  CPU only."""
from __future__ import annotations

import ctypes

import pytest
import torch

from oracle import kv4 as ref
from triton_fused_rmsnorm_qkv import _lib

A = 1 << 32  # fake addresses far apart, never dereferenced: validation fails before any launch


def desc(**kw):
    a = dict(data=A, n_blocks=8, n_kv_heads=2, head_dim=128, block_size=16, group_size=128, dtype=_lib.BF16, reserved=0)
    a.update(kw)
    return _lib.KV4CacheDesc(*(a[name] for name, _ in _lib.KV4CacheDesc._fields_))


def attention(cache=None, **kw):
    a = dict(q=2 * A, q_r=1024, q_t=1024, q_h=128, n_q=8, start=3 * A, T=4, S=0, R=2, bound=2, table=4 * A, stride=9,
             width=9, lens=5 * A, window=0, scale=1.0, out=6 * A, o_t=1024, ws=7 * A, ws_bytes=1 << 30, flags=0,
             stream=None)
    a.update(kw)
    d = desc(**(cache or {}))
    _lib.load()
    return _lib.kv4["attention"](ctypes.addressof(d), *a.values())


@pytest.mark.parametrize("cache,kw,code", [
    (dict(data=0), {}, _lib.ERR_NULL),
    (dict(dtype=_lib.F32), {}, _lib.ERR_DTYPE),
    (dict(head_dim=96), {}, _lib.ERR_SHAPE),
    (dict(head_dim=64), {}, _lib.ERR_SHAPE),            # group 128 > head_dim
    (dict(group_size=16), {}, _lib.ERR_SHAPE),
    (dict(block_size=24), {}, _lib.ERR_SHAPE),
    (dict(block_size=0), {}, _lib.ERR_SHAPE),
    (dict(n_blocks=0), {}, _lib.ERR_SHAPE),
    (dict(n_blocks=1 << 28), {}, _lib.ERR_SHAPE),       # 2^32 slots
    (dict(n_kv_heads=0), {}, _lib.ERR_SHAPE),
    (dict(data=A + 64), {}, _lib.ERR_ALIGN),
    ({}, dict(q=None), _lib.ERR_NULL),
    ({}, dict(out=None), _lib.ERR_NULL),
    ({}, dict(table=None), _lib.ERR_NULL),
    ({}, dict(lens=None), _lib.ERR_NULL),
    ({}, dict(T=0), _lib.ERR_SHAPE),
    ({}, dict(R=0), _lib.ERR_SHAPE),
    ({}, dict(start=None, S=0), _lib.ERR_SHAPE),
    ({}, dict(start=None, S=3), _lib.ERR_SHAPE),
    ({}, dict(n_q=9), _lib.ERR_SHAPE),
    ({}, dict(bound=-1), _lib.ERR_SHAPE),
    ({}, dict(window=-1), _lib.ERR_SHAPE),
    ({}, dict(stride=8), _lib.ERR_SHAPE),
    ({}, dict(scale=0.0), _lib.ERR_SHAPE),
    ({}, dict(scale=float("nan")), _lib.ERR_SHAPE),
    ({}, dict(scale=float("inf")), _lib.ERR_SHAPE),
    ({}, dict(o_t=1000), _lib.ERR_SHAPE),
    ({}, dict(q_h=-128), _lib.ERR_SHAPE),
    ({}, dict(q=2 * A + 2), _lib.ERR_ALIGN),
    ({}, dict(q_t=1025), _lib.ERR_ALIGN),
    ({}, dict(out=6 * A + 8), _lib.ERR_ALIGN),
    ({}, dict(out=2 * A + 1024), _lib.ERR_ALIAS),
    ({}, dict(ws=None), _lib.ERR_WORKSPACE),
    ({}, dict(ws_bytes=4096), _lib.ERR_WORKSPACE),
    ({}, dict(ws=7 * A + 16), _lib.ERR_ALIGN),
    ({}, dict(flags=64), _lib.ERR_SCHEDULE),
])
def test_attention_rejects(cache, kw, code):
    assert attention(cache, **kw) == code
    assert _lib.last_error() != ""


@pytest.mark.parametrize("kw,code", [
    (dict(k=None), _lib.ERR_NULL), (dict(slots=None), _lib.ERR_NULL), (dict(B=0), _lib.ERR_SHAPE),
    (dict(S=0), _lib.ERR_SHAPE), (dict(B=1 << 20, S=1 << 20), _lib.ERR_SHAPE), (dict(k=2 * A + 4), _lib.ERR_ALIGN),
    (dict(ks=129), _lib.ERR_ALIGN), (dict(flags=2), _lib.ERR_SCHEDULE),
])
def test_append_rejects(kw, code):
    a = dict(k=2 * A, v=3 * A, B=1, S=4, kb=0, ks=256, kh=128, vb=0, vs=256, vh=128, slots=4 * A, flags=0, stream=None)
    a.update(kw)
    d = desc()
    _lib.load()
    assert _lib.kv4["append"](ctypes.addressof(d), *a.values()) == code


@pytest.mark.parametrize("kw,code", [
    (dict(slots=None), _lib.ERR_NULL), (dict(T=0), _lib.ERR_SHAPE), (dict(v=3 * A + 8), _lib.ERR_ALIGN),
    (dict(flags=4), _lib.ERR_SCHEDULE),
])
def test_gather_rejects(kw, code):
    a = dict(slots=2 * A, T=4, k=4 * A, v=3 * A, flags=0, stream=None)
    a.update(kw)
    d = desc()
    _lib.load()
    assert _lib.kv4["gather"](ctypes.addressof(d), *a.values()) == code


@pytest.mark.parametrize("kw,code", [
    (dict(ctx=None), _lib.ERR_NULL), (dict(slots=None), _lib.ERR_NULL), (dict(free=None), _lib.ERR_NULL),
    (dict(R=0), _lib.ERR_SHAPE), (dict(T=-1), _lib.ERR_SHAPE), (dict(block=12), _lib.ERR_SHAPE),
    (dict(stride=3), _lib.ERR_SHAPE), (dict(n_free_out=5 * A), _lib.ERR_ALIAS), (dict(flags=8), _lib.ERR_SCHEDULE),
])
def test_plan_rejects(kw, code):
    a = dict(ctx=A, new=2 * A, R=2, table=3 * A, stride=4, width=4, free=4 * A, cap=10, n_free=5 * A, block=16, T=8,
             start=6 * A, positions=7 * A, slots=8 * A, lens=9 * A, n_free_out=10 * A, refused=11 * A, flags=0,
             stream=None)
    a.update(kw)
    _lib.load()
    assert _lib.kv4["plan"](*a.values()) == code


def test_sizes():
    lib = _lib.load()
    assert lib.fqkv_kv4_record_bytes(128, 128) == 2176 and lib.fqkv_kv4_record_bytes(64, 32) == 1280
    assert lib.fqkv_kv4_record_bytes(96, 32) == 0 and lib.fqkv_kv4_record_bytes(64, 128) == 0
    assert lib.fqkv_kv4_workspace_bytes(32, 8, 128, 1) > 4096
    assert lib.fqkv_kv4_workspace_bytes(30, 8, 128, 1) == -_lib.ERR_SHAPE


@pytest.mark.parametrize("D,group", [(128, 128), (128, 32), (64, 64)])
def test_code_places_are_a_bijection(D, group):
    places = {ref.code_place(kind, t, d, D) for kind in "kv" for t in range(16) for d in range(D)}
    assert len(places) == 2 * 16 * D and {p[0] for p in places} == set(range(16 * D))


def test_quantiser_error_is_at_most_half_a_step():
    x = torch.randn(50, 128).to(torch.bfloat16)
    code, scale, low = ref.quantise(x, 32)
    err = (ref.values(code, scale, low) - x.double()).abs().unflatten(-1, (-1, 32)).amax(-1)
    # half a step, and 15 times the rounding of the scale where the maximum is cut off
    assert (err <= scale.double() * (0.5 + 15 * 2.0 ** -8)).all()
