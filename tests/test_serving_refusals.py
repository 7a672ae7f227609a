"""Rotary positions, the paged cache and attention over it: argument checks, in Python and at the C
boundary, before any CUDA call."""
import ctypes

import pytest
import torch

import natten_b200 as nb
import natten_b200._lib as L


def _x(*shape, dtype=torch.bfloat16):
    return torch.zeros(*shape, dtype=dtype)


def _cache(pages=4, page=8, heads=2, dim=16, dtype=torch.bfloat16):
    return nb.KVCache.allocate(pages, page, heads, dim, dtype, device="cpu")


def _i32(*v):
    return torch.tensor(v, dtype=torch.int32)


def test_default_channels_of_the_axes():
    assert nb.rotary_axis_dims(128, 3) == (48, 40, 40)
    assert nb.rotary_axis_dims(64, 2) == (32, 32)
    assert nb.rotary_axis_dims(64, 1) == (64,)
    assert nb.rotary_axis_dims(16, 3) == (6, 6, 4)
    assert nb.rotary_axis_dims(7, 1) == (6,)
    assert nb.rotary_axis_dims(1, 2) == (0, 0)


@pytest.mark.parametrize("error,args,kw", [
    (ValueError, (_x(2, 4, 16),), {}),
    (ValueError, (_x(2, 4, 1, 16, dtype=torch.float64),), {}),
    (ValueError, (_x(2, 4, 1, 16), _x(2, 5, 1, 16)), {}),
    (ValueError, (_x(2, 4, 1, 16), _x(2, 4, 1, 8)), {}),
    (ValueError, (_x(2, 4, 1, 16), _x(2, 4, 1, 16, dtype=torch.float16)), {}),
    (NotImplementedError, (_x(2, 4, 1, 264),), {}),
    (ValueError, (_x(2, 4, 1, 16),), {"axis_dims": (18,)}),
    (ValueError, (_x(2, 4, 1, 16),), {"axis_dims": (7,)}),
    (ValueError, (_x(2, 4, 1, 16),), {"axis_dims": (8, 8)}),
    (ValueError, (_x(2, 4, 4, 1, 16),), {"theta": 0.0}),
    (ValueError, (_x(2, 4, 4, 1, 16),), {"theta": (1e4, float("inf"))}),
    (ValueError, (_x(2, 4, 4, 1, 16),), {"position_scale": float("nan")}),
    (ValueError, (_x(2, 4, 4, 1, 16),), {"origin": (1, 2, 3)}),
    (ValueError, (_x(2, 4, 4, 1, 16),), {"origin": 1.5}),
    (ValueError, (_x(2, 4, 1, 16),), {"interleaved": 1}),
    (ValueError, (_x(2, 4, 1, 16),), {"positions": _x(2, 4, 1)}),
    (ValueError, (_x(2, 4, 1, 16),), {"positions": torch.zeros(2, 5, 1, dtype=torch.int32)}),
    (ValueError, (_x(3, 4, 1, 16),), {"positions": torch.zeros(2, 4, 1, dtype=torch.int32)}),
    (ValueError, (_x(2, 4, 1, 16),), {"positions": torch.zeros(2, 4, 4, dtype=torch.int32)}),
    (ValueError, (_x(2, 4, 1, 16),), {"positions": torch.zeros(2, 4, 1, dtype=torch.int32), "origin": 2}),
    (RuntimeError, (_x(2, 4, 1, 16),), {}),                       # CPU tensors
])
def test_rotary_refuses(error, args, kw):
    with pytest.raises(error):
        nb.rotary(*args, **kw)


def test_cache_refusals():
    c, t, n = _cache(), torch.zeros(2, 3, dtype=torch.int32), _i32(3, 4)
    kv = _x(2, 1, 2, 16)
    bad_caches = [
        nb.KVCache(c.key, c.value[:, :4]),
        nb.KVCache(c.key, c.value.half()),
        nb.KVCache(c.key.double(), c.value.double()),
        nb.KVCache(c.key.transpose(1, 3), c.value.transpose(1, 3)),
        nb.KVCache(c.key.to(torch.float8_e4m3fn), c.value.to(torch.float8_e4m3fn)),
        nb.KVCache(c.key, c.value, torch.zeros(4, 8, 2), torch.zeros(4, 8, 2)),
        nb.KVCache(c.key[:, :0], c.value[:, :0]),
        (c.key, c.value),
        nb.KVCache(c.key, None),
    ]
    for bad in bad_caches:
        for call in (lambda: nb.kv_cache_write(bad, kv, kv, t), lambda: nb.kv_cache_read(bad, t, 3),
                     lambda: nb.na1d_decode(kv, bad, t, n)):
            with pytest.raises(ValueError):
                call()
    wide = _cache(dim=264)
    with pytest.raises(NotImplementedError):
        nb.kv_cache_read(wide, t, 3)
    with pytest.raises(ValueError):
        nb.KVCache.allocate(4, 8, 2, 16, torch.float8_e5m2, device="cpu")
    for call in (
            lambda: nb.kv_cache_write(c, _x(2, 1, 3, 16), _x(2, 1, 3, 16), t),      # heads
            lambda: nb.kv_cache_write(c, _x(2, 1, 2, 8), _x(2, 1, 2, 8), t),        # channels
            lambda: nb.kv_cache_write(c, kv, _x(2, 2, 2, 16), t),
            lambda: nb.kv_cache_write(c, kv.half(), kv.half(), t),                  # data type
            lambda: nb.kv_cache_write(c, kv, kv, t.long()),
            lambda: nb.kv_cache_write(c, kv, kv, t[:1]),
            lambda: nb.kv_cache_write(c, kv, kv, t, n.long()),
            lambda: nb.kv_cache_write(c, kv, kv, t, _i32(1)),
            lambda: nb.kv_cache_write(c, kv, kv, t, n, _i32(1, 2, 3)),
            lambda: nb.kv_cache_write(nb.KVCache(c.key[:1].expand(4, -1, -1, -1), c.value), kv, kv, t),
            lambda: nb.kv_cache_read(c, t, -1),
            lambda: nb.kv_cache_read(c, t, 2.0),
            lambda: nb.kv_cache_read(c, t, 3, dtype=torch.float16),
            lambda: nb.kv_cache_read(c, t, 3, counts=_i32(1)),
            lambda: nb.na1d_decode(_x(2, 1, 3, 16), c, t, n),                       # heads
            lambda: nb.na1d_decode(_x(2, 1, 1, 16), c, t, n),
            lambda: nb.na1d_decode(_x(2, 2, 16), c, t, n),
            lambda: nb.na1d_decode(kv.float(), c, t, n),
            lambda: nb.na1d_decode(kv, c, t, None),
            lambda: nb.na1d_decode(kv, c, t, n.long()),
            lambda: nb.na1d_decode(kv, c, t, n, kernel_size=1),
            lambda: nb.na1d_decode(kv, c, t, n, kernel_size=4, dilation=0),
            lambda: nb.na1d_decode(kv, c, t, n, scale=-1.0)):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(NotImplementedError):
        nb.na1d_decode(kv.clone().requires_grad_(), c, t, n)
    with pytest.raises(NotImplementedError):
        nb.kv_cache_write(c, kv.clone().requires_grad_(), kv, t)
    for call in (lambda: nb.kv_cache_write(c, kv, kv, t), lambda: nb.kv_cache_read(c, t, 3),
                 lambda: nb.na1d_decode(kv, c, t, n)):
        with pytest.raises(RuntimeError):          # CPU tensors
            call()


ONE = ctypes.c_void_p(1024)


def _struct(**kw):
    c = L.KvCacheStruct()
    a = dict(key=1024, value=1024, pages=4, page_size=8, heads=2, head_dim=16, dtype=L.BF16)
    a.update(kw)
    for n, v in a.items():
        setattr(c, n, v)
    c.key_stride[:] = c.value_stride[:] = (256, 32, 16)
    return c


def _decode(c, B=2, T=1, Hq=2, dtype=L.BF16, max_pages=3, kernel=0, dilation=1, scale=1.0, query=ONE,
            workspace=ONE, lengths=ONE, table=ONE):
    return L.lib.b200na_na1d_decode(query, L.longs((32, 32, 16)), ctypes.byref(c), ONE, None, B, T, Hq,
                                    dtype, table, 3, max_pages, lengths, kernel, dilation, scale, workspace,
                                    None)


def test_decode_c_entry_refuses():
    assert _decode(_struct(), Hq=3) == L.ERR_INVALID_ARGUMENT
    assert _decode(_struct(head_dim=264)) == L.ERR_UNSUPPORTED
    assert _decode(_struct(), dtype=L.E4M3) == L.ERR_UNSUPPORTED
    assert _decode(_struct(), dtype=L.F16) == L.ERR_INVALID_ARGUMENT
    assert _decode(_struct(dtype=L.E4M3)) == L.ERR_INVALID_ARGUMENT          # no scales
    assert _decode(_struct(), kernel=-1) == L.ERR_INVALID_ARGUMENT
    assert _decode(_struct(), dilation=0) == L.ERR_INVALID_ARGUMENT
    assert _decode(_struct(), scale=0.0) == L.ERR_INVALID_ARGUMENT
    assert _decode(_struct(), scale=float("inf")) == L.ERR_INVALID_ARGUMENT
    assert _decode(_struct(), query=None) == L.ERR_INVALID_ARGUMENT
    # long tables work through ranges of all sequences' keys, which need scratch
    assert _decode(_struct(), workspace=None, max_pages=10000) == L.ERR_INVALID_ARGUMENT
    assert _decode(_struct(), max_pages=2 ** 28) == L.ERR_UNSUPPORTED        # 2^31 tokens
    assert _decode(_struct(), lengths=None) == L.ERR_INVALID_ARGUMENT
    assert _decode(_struct(), table=None) == L.ERR_INVALID_ARGUMENT
    assert _decode(_struct(), workspace=ctypes.c_void_p(1032)) == L.ERR_ALIGNMENT
    assert _decode(_struct(page_size=0)) == L.ERR_INVALID_ARGUMENT
    assert _decode(_struct(key=None)) == L.ERR_INVALID_ARGUMENT
    assert _decode(_struct(), B=0) == L.OK and _decode(_struct(), T=0) == L.OK
    sizes = [L.lib.b200na_na1d_decode_workspace(2, 1, 2, ctypes.byref(_struct()), pages, 0, 1, L.BF16)
             for pages in (3, 10000)]
    assert sizes[0] == 0 and sizes[1] > 0
    assert L.lib.b200na_na1d_decode_workspace(2, 1, 3, ctypes.byref(_struct()), 3, 0, 1,
                                              L.BF16) == L.ERR_INVALID_ARGUMENT


def test_move_and_rotary_c_entries_refuse():
    s3 = L.longs((32, 32, 16))
    w = lambda c, key=ONE, T=1, dtype=L.BF16, strides=s3: L.lib.b200na_kv_cache_write(  # noqa: E731
        ctypes.byref(c), key, ONE, 2, T, dtype, strides, s3, ONE, 3, 3, None, None, None)
    assert w(_struct(), key=None) == L.ERR_INVALID_ARGUMENT
    assert w(_struct(), T=-1) == L.ERR_INVALID_ARGUMENT
    assert w(_struct(), dtype=L.F32) == L.ERR_INVALID_ARGUMENT
    assert w(_struct(), strides=None) == L.ERR_INVALID_ARGUMENT
    assert w(_struct(), T=0) == L.OK and w(_struct(pages=0, key=None, value=None)) == L.OK
    r = lambda c, length=1, dtype=L.BF16: L.lib.b200na_kv_cache_read(  # noqa: E731
        ctypes.byref(c), ONE, None, 2, length, dtype, ONE, 3, 3, None, None, None)
    assert r(_struct()) == L.ERR_INVALID_ARGUMENT
    assert r(_struct(), length=-1) == L.ERR_INVALID_ARGUMENT
    assert r(_struct(), length=0) == L.OK

    def rot(D=16, dims=(16,), theta=(1e4,), axes=1, ndim=1, dtype=L.BF16, positions=None, kind=0,
            q=ONE, shape=(4,), Hkv=0):
        st = L.longs([1] * 5)
        return L.lib.b200na_rotary(q, None, ONE, None, ndim, L.ints(shape), 1, 2, Hkv, D, dtype, st, st, axes,
                                   L.ints(dims), L.doubles(theta), L.doubles([1.0] * 3), L.longs([0] * 3),
                                   positions, kind, 0, 0, 0, None)
    assert rot(q=None) == L.ERR_INVALID_ARGUMENT
    assert rot(Hkv=1) == L.ERR_INVALID_ARGUMENT
    assert rot(dims=(18,)) == L.ERR_INVALID_ARGUMENT
    assert rot(dims=(7,)) == L.ERR_INVALID_ARGUMENT
    assert rot(theta=(0.0,)) == L.ERR_INVALID_ARGUMENT
    assert rot(axes=2, dims=(8, 8), theta=(1e4, 1e4)) == L.ERR_INVALID_ARGUMENT   # axes != ndim
    assert rot(positions=ONE, kind=3) == L.ERR_INVALID_ARGUMENT
    assert rot(dtype=L.E4M3) == L.ERR_UNSUPPORTED
    assert rot(D=264, dims=(264,)) == L.ERR_UNSUPPORTED
    assert rot(ndim=4, shape=(1, 1, 1, 1)) == L.ERR_INVALID_ARGUMENT
    assert rot(shape=(0,)) == L.OK
