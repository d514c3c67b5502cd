"""Attention over packed rows and the 16-bit cache without a GPU: what every entry point refuses (the checks run for CPU
tensors too, the last refuses the device), what the operators write, workspaces, and the C ABI's refusals.  Nothing is
launched."""

import ctypes
import math

import pytest
import torch

from cqgdn import _lib, attention, kvcache, rotary

DEVICE = "requires tensors on a ROCm GPU"
B = torch.bfloat16


def i(*x):
    return torch.zeros(*x, dtype=torch.int32)


def _attend(**kw):
    a = dict(q=torch.zeros(5, 4, 64, dtype=B), k=torch.zeros(7, 2, 64, dtype=B), v=torch.zeros(7, 2, 64, dtype=B), limit=i(5)) | kw
    return attention.attend(a.pop("q"), a.pop("k"), a.pop("v"), a.pop("limit"), **a)


@pytest.mark.parametrize("kw,match", [
    (dict(q=torch.zeros(5, 4, 128, dtype=B)), "head_dim"),
    (dict(q=torch.zeros(5, 64, dtype=B)), "T, heads, head_dim"),
    (dict(v=torch.zeros(6, 2, 64, dtype=B)), "S, kv_heads, head_dim"),
    (dict(k=torch.zeros(7, 2, 64).half()), "share one type"),
    (dict(q=torch.zeros(5, 4, 64)), "bf16 or fp16"),
    (dict(q=torch.zeros(5, 3, 64, dtype=B)), "no multiple"),
    (dict(q=torch.zeros(5, 4, 96, dtype=B), k=torch.zeros(7, 2, 96, dtype=B), v=torch.zeros(7, 2, 96, dtype=B)), "64, 128 or 256"),
    (dict(limit=i(4)), "limit must hold a value a row"),
    (dict(limit=torch.zeros(5, dtype=torch.int64)), "limit must be an int32 vector"),
    (dict(first=i(6)), "first must hold"),
    (dict(positions=torch.zeros(5)), "positions must be an int32 vector"),
    (dict(slopes=torch.zeros(2)), "slopes must hold"),
    (dict(slopes=torch.zeros(4, dtype=B)), "slopes must hold"),
    (dict(slopes=torch.zeros(4, requires_grad=True)), "constants"),
    (dict(cap=0.0), "cap must be positive"),
    (dict(cap=-1.0), "cap must be positive"),
    (dict(cap=math.nan), "cap must be positive"),
    (dict(cap=math.inf), "cap must be positive"),
    (dict(cap=1e300), "cap must be positive"),
    (dict(scale=math.nan), "scale must be finite"),
    (dict(scale=1e300), "scale must be finite"),
    (dict(), DEVICE),
    (dict(q=torch.zeros(5, 4, 64, dtype=B, requires_grad=True)), DEVICE),
    (dict(cap=1e-50), "cap must be positive"),  # 0 in fp32
])
def test_attend_refusals(kw, match):
    with pytest.raises(ValueError, match=match):
        _attend(**kw)


@pytest.mark.parametrize("args,kw", [
    (([1, 2],), {}), (([],), {}), (([0, 3, 2],), {}), (([0, 3],), dict(window=0)), (([0, 3],), dict(prefix=(1, 2))),
])
def test_documents_refusals(args, kw):
    with pytest.raises(ValueError):
        attention.documents(*args, device="cpu", **kw)


def test_documents_of_nothing():
    first, limit = attention.documents([0], device="cpu")
    assert first.numel() == limit.numel() == 0 and first.dtype == limit.dtype == torch.int32


def _cache(**kw):
    return kvcache.KVCache.empty(**(dict(pages=3, heads=2, page=16, head_dim=64, bits=16, device="cpu") | kw))


def test_cache_kinds():
    assert _cache().bits == 16 and _cache(bits=4).bits == 4 and kvcache.KVCache.empty(1, 1, device="cpu").bits == 4
    assert _cache().pages == 3 and _cache().heads == 2 and tuple(_cache().data.shape) == (3, 2, 2, 16, 64)
    with pytest.raises(ValueError, match="bits"):
        _cache(bits=8)
    with pytest.raises(ValueError, match="bf16 or fp16 rows"):
        _cache(dtype=torch.float32)
    for bad in (torch.zeros(3, 2, 16, 64, dtype=B), torch.zeros(3, 2, 2, 32, 64, dtype=B), torch.zeros(3, 2, 2, 16, 64).half()):
        with pytest.raises(ValueError, match="data must be"):
            kvcache.KVCache(bad, page=16, head_dim=64)


def _append(**kw):
    a = dict(q=torch.zeros(5, 4, 64, dtype=B), k=torch.zeros(5, 2, 64, dtype=B), v=torch.zeros(5, 2, 64, dtype=B),
             positions=i(1, 5), plan=rotary.plan(32, device="cpu"), slots=i(5), cache=_cache()) | kw
    return kvcache.append(a["cache"], a["q"], a["k"], a["v"], a["positions"], a["plan"], a["slots"])


@pytest.mark.parametrize("kw,match", [
    (dict(q=torch.zeros(5, 4, 64)), "as the cache is"),
    (dict(q=torch.zeros(4, 4, 64, dtype=B)), "q must be"),
    (dict(k=torch.zeros(5, 3, 64, dtype=B), v=torch.zeros(5, 3, 64, dtype=B)), "as the cache is"),
    (dict(v=torch.zeros(5, 2, 128, dtype=B)), "as the cache is"),
    (dict(slots=i(4)), "a value a row"),
    (dict(slots=torch.zeros(5, dtype=torch.int64)), "int32 vector"),
    (dict(positions=i(1, 4)), "positions"),
    (dict(positions=torch.zeros(1, 5)), "positions"),
    (dict(plan=rotary.plan(128, device="cpu")), "the plan turns 128"),
    (dict(plan=rotary.plan(32, sections=(4, 6, 6), device="cpu"), positions=i(2, 5)), "2 axes, the plan 3"),
    (dict(), DEVICE),
    (dict(cache=_cache(bits=4)), DEVICE),
])
def test_append_refusals(kw, match):
    with pytest.raises(ValueError, match=match):
        _append(**kw)


def _cached(**kw):
    a = dict(q=torch.zeros(5, 4, 64, dtype=B), cache=_cache(), tables=i(2, 3), starts=i(3), visible=i(5)) | kw
    return kvcache.attend(a.pop("q"), a.pop("cache"), a.pop("tables"), a.pop("starts"), a.pop("visible"), **a)


@pytest.mark.parametrize("kw,match", [
    (dict(q=torch.zeros(5, 4, 64).half()), "as the cache is"),
    (dict(q=torch.zeros(5, 4, 128, dtype=B)), "as the cache is"),
    (dict(q=torch.zeros(5, 3, 64, dtype=B)), "no multiple"),
    (dict(tables=torch.zeros(2, 3)), "tables"),
    (dict(starts=i(2)), "starts must hold"),
    (dict(visible=i(4)), "starts must hold"),
    (dict(positions=i(4)), "positions must hold"),
    (dict(slopes=torch.zeros(2)), "slopes must hold"),
    (dict(cap=0.0), "cap must be positive"),
    (dict(cap=math.inf), "cap must be positive"),
    (dict(scale=math.inf), "scale must be finite"),
    (dict(window=0), "window"),
    (dict(max_queries=0), "max_queries"),
    (dict(), DEVICE),
])
def test_cached_attend_refusals(kw, match):
    with pytest.raises(ValueError, match=match):
        _cached(**kw)


@pytest.mark.parametrize("kw", [dict(cap=5.0), dict(slopes=torch.zeros(4)), dict(positions=i(5))])
def test_four_bits_take_no_cap_or_bias(kw):
    with pytest.raises(ValueError, match="need a 16-bit cache"):
        _cached(cache=_cache(bits=4), **kw)


def test_read_refusals():
    with pytest.raises(ValueError, match="int32 vector"):
        kvcache.read(_cache(), torch.zeros(3, dtype=torch.int64))


@pytest.mark.parametrize("name,written", [("attend", set()), ("attend_bwd", set()), ("kv16_append", {"data"}), ("kv16_attend", set())])
def test_written_arguments(name, written):
    schema = getattr(_lib.ops(), name).default._schema
    assert {a.name for a in schema.arguments if a.alias_info is not None and a.alias_info.is_write} == written
    assert all(r.alias_info is None for r in schema.returns)


def test_no_gradient_passes_through_the_16_bit_cache():
    _lib.ops()
    lib = torch.library.Library("cqgdn", "IMPL")
    lib.impl("kv16_attend", lambda q, *a: (torch.empty_like(q), torch.empty(0, device="meta")), "Meta")
    lib.impl("kv16_append", lambda q, *a: torch.empty_like(q), "Meta")
    try:
        m = lambda *x: torch.zeros(*x, dtype=torch.int32, device="meta")  # noqa: E731
        cache = kvcache.KVCache(torch.empty(3, 2, 2, 16, 64, dtype=B, device="meta"), page=16, head_dim=64)
        q = torch.empty(4, 4, 64, dtype=B, device="meta", requires_grad=True)
        k = torch.empty(4, 2, 64, dtype=B, device="meta")
        plan = rotary.RotaryPlan(torch.zeros(4, dtype=torch.int64, device="meta"), m(4))
        for out in (kvcache.attend(q, cache, m(2, 3), m(3), m(4)), kvcache.append(cache, q, k, k, m(1, 4), plan, m(4))):
            assert not out.requires_grad
    finally:
        lib._destroy()


# ---- the C ABI ---------------------------------------------------------------------------------------

def test_workspaces_cover_the_parts():
    lib = _lib.lib()
    assert lib.cqgdn_attend_fwd_workspace_size(0, 5, 4, 2, 64) == lib.cqgdn_attend_fwd_workspace_size(5, 5, 4, 3, 64) == 0
    assert lib.cqgdn_attend_fwd_workspace_size(5, 5, 4, 2, 96) == 0
    # 64 rows a block: 1536 bytes for each key head, 16 for all; blocks by 128 rows
    for T, S, hq, hk, D in ((1, 1, 1, 1, 64), (317, 253, 16, 4, 128), (5000, 700, 7, 1, 256), (40000, 40000, 16, 16, 128)):
        blocks = -(-T * (hq // hk) // 128) * 2
        need = lib.cqgdn_attend_bwd_workspace_size(T, S, hq, hk, D)
        assert need >= blocks * (1536 * hk + 16)
        rest = need - (blocks * (1536 * hk + 16) + 255) // 256 * 256
        assert rest % (2 * S * hk * D * 4) == 0
    assert lib.cqgdn_kv16_attend_workspace_size(0, 1, 4, 2, 64, 1, 3, 16) == 0


def test_c_abi_refusals():
    lib = _lib.lib()
    buf = (ctypes.c_char * 4096)()
    p = (ctypes.addressof(buf) + 255) // 256 * 256

    def fwd(**kw):
        a = dict(q=p, qt=256, qh=64, k=p, kt=128, kh=64, v=p, vt=128, vh=64, dtype=0, T=2, S=3, heads=4, kv=2, D=64, first=None,
                 limit=p, positions=None, scale=1.0, cap=0.0, slopes=None, out=p, lse=p, ws=None, n=0, stream=None) | kw
        return lib.cqgdn_attend_fwd(*a.values())

    for kw, rc in ((dict(D=96), _lib.EUNSUPPORTED), (dict(T=-1), _lib.EINVAL), (dict(heads=3), _lib.EINVAL), (dict(dtype=2), _lib.EINVAL),
                   (dict(scale=math.nan), _lib.EINVAL), (dict(cap=-1.0), _lib.EINVAL), (dict(cap=math.inf), _lib.EINVAL),
                   (dict(q=None), _lib.EINVAL), (dict(k=p + 2), _lib.EINVAL), (dict(vt=100), _lib.EINVAL),
                   (dict(kt=1 << 24), _lib.EINVAL), (dict(limit=None), _lib.EINVAL), (dict(out=p + 8), _lib.EINVAL),
                   (dict(T=1 << 26), _lib.EUNSUPPORTED), (dict(S=1 << 27), _lib.EUNSUPPORTED),
                   (dict(T=400, S=5000), _lib.EINVAL),  # parts without a workspace
                   (dict(T=0), _lib.OK)):
        assert fwd(**kw) == rc, (kw, lib.cqgdn_last_error())

    def bwd(**kw):
        a = dict(q=p, qt=256, qh=64, k=p, kt=128, kh=64, v=p, vt=128, vh=64, dy=p, yt=256, yh=64, dtype=0, T=2, S=3, heads=4, kv=2,
                 D=64, first=None, limit=p, positions=None, scale=1.0, cap=0.0, slopes=None, out=p, lse=p, dlse=None, dq=p, dk=p,
                 dv=p, ws=p, n=1, stream=None) | kw
        return lib.cqgdn_attend_bwd(*a.values())

    for kw, rc in ((dict(D=32), _lib.EUNSUPPORTED), (dict(lse=None), _lib.EINVAL), (dict(dy=None), _lib.EINVAL), (dict(dq=None), _lib.EINVAL),
                   (dict(dk=None), _lib.EINVAL), (dict(dv=p + 4), _lib.EINVAL), (dict(), _lib.EINVAL), (dict(ws=None, n=1 << 30), _lib.EINVAL),
                   (dict(T=0, S=0), _lib.OK)):
        assert bwd(**kw) == rc, (kw, lib.cqgdn_last_error())

    def append(**kw):
        a = dict(q=p, qt=256, qh=64, heads=4, k=p, kt=128, kh=64, v=p, vt=128, vh=64, T=2, kv=2, D=64, rotary=32, adjacent=0, dtype=0,
                 positions=p, wide=0, stride=2, axes=1, turns=p, axis=p, slots=p, out=p, data=p, pages=1, page=16, stream=None) | kw
        return lib.cqgdn_kv16_append(*a.values())

    for kw, rc in ((dict(D=80), _lib.EUNSUPPORTED), (dict(page=24), _lib.EINVAL), (dict(rotary=66), _lib.EINVAL), (dict(rotary=3), _lib.EINVAL),
                   (dict(axes=0), _lib.EINVAL), (dict(dtype=2), _lib.EINVAL), (dict(out=None), _lib.EINVAL), (dict(slots=None), _lib.EINVAL),
                   (dict(positions=None), _lib.EINVAL), (dict(data=None), _lib.EINVAL), (dict(pages=1 << 28), _lib.EUNSUPPORTED),
                   (dict(T=1 << 24), _lib.EUNSUPPORTED), (dict(kv=40000), _lib.EUNSUPPORTED), (dict(T=0), _lib.OK)):
        assert append(**kw) == rc, (kw, lib.cqgdn_last_error())

    def cached(**kw):
        a = dict(q=p, qt=256, qh=64, dtype=0, T=2, heads=4, D=64, data=p, pages=1, page=16, kv=2, tables=p, ts=3, columns=3, starts=p,
                 N=1, visible=p, window=0, positions=None, scale=1.0, cap=0.0, slopes=None, most=1, out=p, lse=None, ws=None, n=0,
                 stream=None) | kw
        return lib.cqgdn_kv16_attend(*a.values())

    for kw, rc in ((dict(D=32), _lib.EUNSUPPORTED), (dict(page=8), _lib.EINVAL), (dict(dtype=2), _lib.EINVAL), (dict(cap=-2.0), _lib.EINVAL),
                   (dict(ts=2), _lib.EINVAL), (dict(most=0), _lib.EINVAL), (dict(window=-1), _lib.EINVAL), (dict(q=p + 2), _lib.EINVAL),
                   (dict(tables=None), _lib.EINVAL), (dict(visible=None), _lib.EINVAL), (dict(T=1 << 26), _lib.EUNSUPPORTED),
                   (dict(columns=1000, ts=1000), _lib.EINVAL),  # parts without a workspace
                   (dict(T=0), _lib.OK)):
        assert cached(**kw) == rc, (kw, lib.cqgdn_last_error())


@pytest.mark.parametrize("kw,rc", [
    (dict(cap=1e-39), _lib.EINVAL), (dict(cap=3e38), _lib.EINVAL), (dict(scale=3e38), _lib.EINVAL), (dict(scale=1e20, cap=1e-19), _lib.EINVAL),
    (dict(S=(1 << 24) + 1, kv=1, slopes=True), _lib.EUNSUPPORTED),
])
def test_scores_that_fp32_does_not_hold(kw, rc):
    lib = _lib.lib()
    buf = (ctypes.c_char * 4096)()
    p = (ctypes.addressof(buf) + 255) // 256 * 256
    if kw.get("slopes"):
        kw = kw | dict(slopes=p)
    a = dict(q=p, qt=256, qh=64, k=p, kt=128, kh=64, v=p, vt=128, vh=64, dtype=0, T=2, S=3, heads=4, kv=2, D=64, first=None,
             limit=p, positions=None, scale=1.0, cap=0.0, slopes=None, out=p, lse=p, ws=None, n=0, stream=None) | kw
    assert lib.cqgdn_attend_fwd(*a.values()) == rc
    back = dict(list(a.items())[:9]) | dict(dy=p, yt=256, yh=64) | dict(list(a.items())[9:21]) | dict(
        out=p, lse=p, dlse=None, dq=p, dk=p, dv=p, ws=p, n=1, stream=None)
    assert lib.cqgdn_attend_bwd(*back.values()) == rc
