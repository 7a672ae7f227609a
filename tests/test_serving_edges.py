"""The serving operators at the edges of what they accept, on the host: sizes and strides at the C boundary and in
the Python checks, before any CUDA call."""
import ctypes
import os
import subprocess
import sys

import pytest
import torch

import natten_b200 as nb
import natten_b200._lib as L


def _cache(pages=4, page_size=8, heads=1, head_dim=1, dtype=L.BF16, **strides):
    c = L.KvCacheStruct()
    for n, v in dict(key=1024, value=1024, pages=pages, page_size=page_size, heads=heads, head_dim=head_dim,
                     dtype=dtype).items():
        setattr(c, n, v)
    for n in ("key_stride", "value_stride", "key_scale_stride", "value_scale_stride"):
        getattr(c, n)[:] = strides.get(n, (page_size * heads * head_dim, heads * head_dim, head_dim))
    return c


def _workspace(c, T=1, Hq=1, max_pages=3, kernel=0, dilation=1, dtype=L.BF16):
    return L.lib.b200na_na1d_decode_workspace(1, T, Hq, ctypes.byref(c), max_pages, kernel, dilation, dtype)


def test_decode_counts_the_rows_of_very_many_tokens_in_64_bits():
    """2^31 - 1 tokens are rounded up to whole items without wrapping around: more rows than a launch has are
    refused, for every kernel."""
    for T in (2 ** 31 - 1, 2 ** 31 - 7):
        for c, dtype in ((_cache(), L.BF16), (_cache(head_dim=64), L.BF16), (_cache(head_dim=64, dtype=L.F32), L.F32)):
            assert _workspace(c, T=T, dtype=dtype) == L.ERR_INVALID_ARGUMENT
            assert _workspace(c, T=T, Hq=5, dtype=dtype) == L.ERR_INVALID_ARGUMENT
    # one row an item (dilated, a query head for each key head): as many as fit 31 bits, if their keys do too
    assert _workspace(_cache(), T=2 ** 31 - 1, dilation=2) >= 0
    assert _workspace(_cache(page_size=2 ** 29), T=2 ** 31 - 1, dilation=2) == L.ERR_INVALID_ARGUMENT


def test_caches_whose_places_run_backwards_are_refused():
    """Strides count from the first place of the pool upwards; the stride of an axis with one entry is not
    looked at."""
    ptr, rows = ctypes.c_void_p(1024), L.longs((1, 1, 1))
    for name in ("key_stride", "value_stride", "key_scale_stride", "value_scale_stride"):
        for axis in range(3):
            strides = [64, 8, 4]
            strides[axis] *= -1
            c = _cache(heads=2, dtype=L.E4M3, **{name: strides})
            c.key_scale = c.value_scale = 1024
            calls = (
                lambda: _workspace(c, Hq=2),
                lambda: L.lib.b200na_kv_cache_write(ctypes.byref(c), ptr, ptr, 1, 0, L.BF16, rows, rows, ptr, 3, 3,
                                                    None, None, None),
                lambda: L.lib.b200na_kv_cache_read(ctypes.byref(c), ptr, ptr, 1, 0, L.BF16, ptr, 3, 3, None, None,
                                                   None))
            assert [f() for f in calls] == [L.ERR_INVALID_ARGUMENT] * 3
            c.pages, c.page_size, c.heads = ((1, 8, 2), (4, 1, 2), (4, 8, 1))[axis]
            assert [f() for f in calls] == [L.OK] * 3


def test_sizes_beyond_31_bits_are_refused():
    """Expanded tensors reach them without memory. (The C boundary takes 32-bit sizes: 2^32 + 3 is 3 there.)"""
    far = 2 ** 32 + 3
    x = torch.zeros(1, 1, 1, 2, dtype=torch.bfloat16)
    cache = nb.KVCache.allocate(4, 8, 1, 2, device="cpu")
    table, n = torch.zeros(1, 3, dtype=torch.int32), torch.tensor([3], dtype=torch.int32)
    tokens, heads, batch = x.expand(1, far, 1, 2), x.expand(1, 1, far, 2), x.expand(far, 1, 1, 2)
    wide = nb.KVCache(*(torch.zeros(1, 1, 1, 2, dtype=torch.bfloat16).expand(1, far, 1, 2) for _ in range(2)))
    for call in (
            lambda: nb.kv_cache_write(cache, tokens, tokens, table),
            lambda: nb.kv_cache_write(cache, batch, batch, table.expand(far, 3)),
            lambda: nb.kv_cache_read(cache, table.expand(far, 3), 1),
            lambda: nb.kv_cache_read(cache, table[:, :1].expand(1, far), 1),
            lambda: nb.kv_cache_read(wide, table, 1),
            lambda: nb.na1d_decode(tokens, cache, table, n),
            lambda: nb.na1d_decode(heads, cache, table, n),
            lambda: nb.na1d_decode(batch, cache, table.expand(far, 3), n.expand(far)),
            lambda: nb.rotary(x, heads), lambda: nb.rotary(heads), lambda: nb.rotary(tokens, tokens)):
        with pytest.raises(NotImplementedError):
            call()


def test_rotary_does_not_detach_without_registered_operators():
    """NATTEN_B200_DISABLE_TORCH_OPS=1 leaves no place for a gradient formula: the call says so."""
    code = ("import torch, natten_b200 as nb\n"
            "x = torch.zeros(1, 4, 2, 16)\n"
            "for args in ((x.clone().requires_grad_(),), (x, x.clone().requires_grad_())):\n"
            "    try:\n"
            "        nb.rotary(*args)\n"
            "    except NotImplementedError as e:\n"
            "        print('refused', 'NATTEN_B200_DISABLE_TORCH_OPS' in str(e))\n"
            "    with torch.no_grad():\n"
            "        try:\n"
            "            nb.rotary(*args)\n"
            "        except RuntimeError as e:\n"
            "            print(type(e).__name__)\n")
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    done = subprocess.run([sys.executable, "-c", code], cwd=root, capture_output=True, text=True, timeout=300,
                          env={**os.environ, "NATTEN_B200_DISABLE_TORCH_OPS": "1"})
    assert done.returncode == 0, done.stderr
    assert done.stdout.split("\n")[:-1] == ["refused True", "RuntimeError"] * 2      # (CPU tensors without gradients)
