"""The attention layers' operators without a GPU: the rotary plan, the refusals of every operator (their
checks run for CPU tensors too, the last refuses the device) and of the C ABI.  Nothing is launched."""

import ctypes
import math

import pytest
import torch

from cqgdn import _lib, kvcache, rotary

DEVICE = "requires tensors on a ROCm GPU"


def test_plan_frequencies_sections_and_order():
    p = rotary.plan(64, theta=1e6, sections=(8, 12, 12), device="cpu")
    for i, t in enumerate(p.turns.tolist()):
        exact = 1e6 ** (-2 * i / 64) / (2 * math.pi) * 2.0 ** 64
        assert abs(t - exact) <= 2 ** 11 + exact * 2 ** -50
    assert p.axis.tolist() == [0] * 8 + [1] * 12 + [2] * 12 and not p.adjacent
    mixed = rotary.plan(16, sections=(2, 3, 3), mixed=True, adjacent=True, device="cpu")
    assert mixed.axis.tolist() == [0, 1, 2, 0, 1, 2, 1, 2] and mixed.adjacent
    assert rotary.plan(2, device="cpu").axis.tolist() == [0]


@pytest.mark.parametrize("kw", [dict(rotary_dim=0), dict(rotary_dim=7), dict(rotary_dim=8, sections=(1, 2)),
                                dict(rotary_dim=8, sections=(5, -1)), dict(rotary_dim=8, sections=()),
                                dict(rotary_dim=8, theta=1.0), dict(rotary_dim=8, theta=math.inf),
                                dict(rotary_dim=8, theta=math.nan)])
def test_plan_refusals(kw):
    with pytest.raises(ValueError):
        rotary.plan(device="cpu", **kw)


def _rotary(**kw):
    p = rotary.plan(kw.pop("rotary_dim", 8), device="cpu")
    a = dict(q=torch.zeros(3, 2, 8), k=torch.zeros(3, 1, 8), positions=torch.zeros(1, 3, dtype=torch.int32)) | kw
    return rotary.rotate(a["q"], a["k"], a["positions"], p)


@pytest.mark.parametrize("kw,match", [
    (dict(q=torch.zeros(4, 2, 8)), "one T and D"),
    (dict(k=torch.zeros(3, 1, 16)), "one T and D"),
    (dict(k=torch.zeros(3, 8)), "T, heads, D"),
    (dict(k=torch.zeros(3, 1, 8).bfloat16()), "share one type"),
    (dict(q=torch.zeros(3, 2, 8).double(), k=torch.zeros(3, 1, 8).double()), "share one type"),
    (dict(positions=torch.zeros(1, 4, dtype=torch.int32)), "positions"),
    (dict(positions=torch.zeros(1, 3)), "positions"),
    (dict(positions=torch.zeros(0, 3, dtype=torch.int32)), "positions"),
    (dict(rotary_dim=10), "the plan turns 10"),
    (dict(), DEVICE),
])
def test_rotate_refusals(kw, match):
    with pytest.raises(ValueError, match=match):
        _rotary(**kw)


def _pages(**kw):
    i = lambda *x: torch.zeros(*x, dtype=torch.int32)  # noqa: E731
    a = dict(cached=i(2), new=i(2), tables=i(2, 4), free=i(8), free_count=i(1), page=16, tokens=5) | kw
    return kvcache.step_pages(**a)


@pytest.mark.parametrize("kw,match", [
    (dict(cached=torch.zeros(2)), "cached must be an int32 vector"),
    (dict(new=torch.zeros(2, dtype=torch.int64)), "new must be an int32 vector"),
    (dict(new=torch.zeros(3, dtype=torch.int32)), "a value a request"),
    (dict(free_count=torch.zeros(2, dtype=torch.int32)), "free_count"),
    (dict(tables=torch.zeros(3, 4, dtype=torch.int32)), "tables"),
    (dict(tables=torch.zeros(4, 2, dtype=torch.int32).t()), "unit column stride"),
    (dict(tables=torch.zeros(1, 4, dtype=torch.int32).expand(2, 4)), "tables"),
    (dict(cached=torch.zeros(4, dtype=torch.int32)[::2]), "contiguous"),
    (dict(page=8), "power of two"),
    (dict(page=48), "power of two"),
    (dict(tokens=-1), "tokens"),
    (dict(), DEVICE),
])
def test_step_pages_refusals(kw, match):
    with pytest.raises(ValueError, match=match):
        _pages(**kw)


def _cache(page=16, d=64, heads=2, pages=3, dtype=torch.bfloat16):
    return kvcache.KVCache.empty(pages, heads, page=page, head_dim=d, dtype=dtype, device="cpu")


def test_cache_layout_and_refusals():
    c = _cache(32, 128)
    assert c.pages == 3 and c.heads == 2 and c.data.shape[2] == 32 * 136
    assert _lib.lib().cqgdn_kv4_page_bytes(32, 128) == 32 * 136 and _lib.lib().cqgdn_kv4_page_bytes(33, 128) == 0
    for kw in (dict(dtype=torch.float32), dict(head_dim=96), dict(page=24), dict(page=8)):
        with pytest.raises(ValueError):
            kvcache.KVCache.empty(3, 2, device="cpu", **kw)
    with pytest.raises(ValueError):
        kvcache.KVCache(c.data[..., :-1], page=32, head_dim=128)
    with pytest.raises(ValueError):
        kvcache.KVCache(c.data.char(), page=32, head_dim=128)


@pytest.mark.parametrize("kw,match", [
    (dict(k=torch.zeros(4, 2, 64)), "as the cache is"),
    (dict(k=torch.zeros(4, 2, 64).half()), "as the cache is"),
    (dict(v=torch.zeros(5, 2, 64).bfloat16()), "k and v must be"),
    (dict(k=torch.zeros(4, 3, 64).bfloat16(), v=torch.zeros(4, 3, 64).bfloat16()), "3 heads, the cache 2"),
    (dict(k=torch.zeros(4, 2, 128).bfloat16(), v=torch.zeros(4, 2, 128).bfloat16()), "data must be"),
    (dict(slots=torch.zeros(3, dtype=torch.int32)), "a value a row"),
    (dict(slots=torch.zeros(4, dtype=torch.int64)), "int32 vector"),
    (dict(), DEVICE),
])
def test_write_refusals(kw, match):
    a = dict(k=torch.zeros(4, 2, 64).bfloat16(), v=torch.zeros(4, 2, 64).bfloat16(),
             slots=torch.zeros(4, dtype=torch.int32)) | kw
    with pytest.raises(ValueError, match=match):
        kvcache.write(_cache(), a["k"], a["v"], a["slots"])


def test_read_refusals():
    with pytest.raises(ValueError, match="int32 vector"):
        kvcache.read(_cache(), torch.zeros(2, 2, dtype=torch.int32))
    with pytest.raises(ValueError, match=DEVICE):
        kvcache.read(_cache(), torch.zeros(2, dtype=torch.int32))


@pytest.mark.parametrize("kw,match", [
    (dict(q=torch.zeros(4, 4, 64)), "as the cache is"),
    (dict(q=torch.zeros(4, 4, 128).bfloat16()), "as the cache is"),
    (dict(q=torch.zeros(4, 64).bfloat16()), "q must be"),
    (dict(q=torch.zeros(4, 3, 64).bfloat16()), "no multiple"),
    (dict(tables=torch.zeros(2, 3)), "tables must be int32"),
    (dict(tables=torch.zeros(3, dtype=torch.int32)), "tables must be int32"),
    (dict(starts=torch.zeros(2, dtype=torch.int32)), "starts must hold"),
    (dict(visible=torch.zeros(5, dtype=torch.int32)), "visible a value a row"),
    (dict(visible=torch.zeros(4, dtype=torch.int64)), "visible must be an int32"),
    (dict(window=0), "window must be positive"),
    (dict(window=-3), "window must be positive"),
    (dict(max_queries=0), "max_queries must be positive"),
    (dict(), DEVICE),
])
def test_attend_refusals(kw, match):
    a = dict(q=torch.zeros(4, 4, 64).bfloat16(), cache=_cache(), tables=torch.zeros(2, 3, dtype=torch.int32),
             starts=torch.zeros(3, dtype=torch.int32), visible=torch.zeros(4, dtype=torch.int32)) | kw
    with pytest.raises(ValueError, match=match):
        kvcache.attend(**a)


P, ODD = ctypes.c_void_p(256), ctypes.c_void_p(264)


def test_c_abi_rotary_rejects_before_launch():
    lib = _lib.lib()

    def call(**kw):
        a = dict(q=P, qt=64, qh=64, hq=1, k=P, kt=64, kh=64, hk=1, T=2, D=64, rot=64, adj=0, back=0, dtype=0, pos=P,
                 wide=0, stride=2, axes=1, turns=P, axis=P, qo=P, ko=P, st=None) | kw
        return lib.cqgdn_rotary(*a.values())

    for kw in (dict(T=-1), dict(D=63), dict(rot=66), dict(rot=3), dict(axes=0), dict(hq=-1), dict(dtype=3),
               dict(q=None), dict(ko=None), dict(pos=None), dict(turns=None)):
        assert call(**kw) == _lib.EINVAL, kw
    assert call(T=1 << 24) == _lib.EUNSUPPORTED and call(hq=65535) == _lib.EUNSUPPORTED
    assert call(T=0) == _lib.OK and call(hq=0, hk=0) == _lib.OK


def test_c_abi_pages_rejects_before_launch():
    lib = _lib.lib()

    def call(**kw):
        a = dict(cached=P, fresh=P, N=2, tables=P, stride=4, columns=4, pool=P, size=8, count=P, page=16, T=3, s=P, l=P,
                 ad=P, c=P, sl=P, po=P, vi=P, st=None) | kw
        return lib.cqgdn_step_pages(*a.values())

    for kw in (dict(N=-1), dict(columns=-1), dict(stride=3), dict(size=-1), dict(T=-1), dict(page=15), dict(cached=None),
               dict(tables=None), dict(pool=None), dict(count=None), dict(s=None), dict(sl=None)):
        assert call(**kw) == _lib.EINVAL, kw
    for kw in (dict(N=1 << 20, columns=1 << 12, stride=1 << 12), dict(size=1 << 28), dict(T=(1 << 31) - 1)):
        assert call(**kw) == _lib.EUNSUPPORTED, kw


def test_c_abi_cache_rejects_before_launch():
    lib = _lib.lib()

    def write(**kw):
        a = dict(k=P, kt=128, kh=128, v=P, vt=128, vh=128, dtype=0, slots=P, T=3, heads=1, D=128, data=P, pages=4,
                 page=16, st=None) | kw
        return lib.cqgdn_kv4_write(*a.values())

    for kw in (dict(k=None), dict(v=ODD), dict(kt=100), dict(dtype=2), dict(T=-1), dict(heads=0), dict(page=20),
               dict(data=None), dict(data=ODD), dict(slots=None), dict(pages=-1)):
        assert write(**kw) == _lib.EINVAL, kw
    for kw in (dict(D=96), dict(pages=1 << 27), dict(T=1 << 30)):
        assert write(**kw) == _lib.EUNSUPPORTED, kw
    assert write(T=0) == _lib.OK

    def read(**kw):
        a = dict(data=P, pages=4, page=16, heads=1, D=128, slots=P, T=3, dtype=0, k=P, v=P, st=None) | kw
        return lib.cqgdn_kv4_read(*a.values())

    for kw in (dict(k=None), dict(v=ODD), dict(dtype=2), dict(slots=None), dict(T=-1)):
        assert read(**kw) == _lib.EINVAL, kw


def test_c_abi_attend_rejects_before_launch():
    lib = _lib.lib()
    need = lib.cqgdn_kv4_attend_workspace_size(3, 2, 4, 2, 128, 2, 64, 16)
    assert need >= 3 * 4 * 2 * 130 * 4  # the positions are split where few requests come
    assert lib.cqgdn_kv4_attend_workspace_size(0, 2, 4, 2, 128, 2, 64, 16) == 0

    def call(**kw):
        a = dict(q=P, qt=512, qh=128, dtype=0, T=3, heads=4, D=128, data=P, pages=4, page=16, kv=2, tables=P, stride=64,
                 columns=64, starts=P, N=2, visible=P, window=0, scale=0.1, most=2, out=P, lse=None, ws=P, size=need,
                 st=None) | kw
        return lib.cqgdn_kv4_attend(*a.values())

    for kw in (dict(q=None), dict(q=ODD), dict(qt=100), dict(T=-1), dict(heads=3), dict(kv=0), dict(page=8),
               dict(stride=63), dict(N=-1), dict(window=-1), dict(scale=math.nan), dict(scale=math.inf), dict(most=0),
               dict(out=None), dict(starts=None), dict(visible=None), dict(tables=None), dict(ws=None),
               dict(size=need - 1), dict(ws=ODD), dict(dtype=2), dict(data=None)):
        assert call(**kw) == _lib.EINVAL, kw
    for kw in (dict(D=32), dict(T=1 << 26), dict(N=1 << 23)):
        assert call(**kw) == _lib.EUNSUPPORTED, kw
    assert call(T=0) == _lib.OK
