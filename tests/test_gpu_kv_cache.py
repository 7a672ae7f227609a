"""Writing the paged key/value cache and reading it back, against plain 64-bit forms."""
import math

import pytest
import torch

import natten_b200 as nb
import serving_reference as ref
from natten_b200 import ops

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.float16, torch.bfloat16]
E4M3 = torch.float8_e4m3fn


def _filled(pages, page, heads, dim, dtype):
    """A cache with something in every place."""
    c = nb.KVCache.allocate(pages, page, heads, dim, dtype)
    for t in c:
        if t is not None:
            t.copy_(torch.randn(t.shape, device="cuda").abs().to(t.dtype) + 1.0 if t.dtype != E4M3
                    else (torch.randn(t.shape, device="cuda") + 2.0).to(E4M3))
    return c


def _bits(t):
    return t.view({1: torch.uint8, 2: torch.int16, 4: torch.int32}[t.element_size()])


def _clone(c):
    return nb.KVCache(*(None if t is None else t.clone() for t in c))


def _check_write(before, after, key, value, table, start, counts):
    """Every written row is right, every other place keeps its bits."""
    table, start, counts = table.cpu(), start.tolist(), counts.tolist()
    pages, ps = before.key.shape[:2]
    touched = torch.zeros(pages, ps, dtype=torch.bool)
    scaled = before.key.dtype == E4M3
    for b in range(key.shape[0]):
        for t in range(min(counts[b], key.shape[1])):
            p = start[b] + t
            if p < 0 or p // ps >= table.shape[1]:
                continue
            page, slot = int(table[b, p // ps]), p % ps
            if not 0 <= page < pages:
                continue
            touched[page, slot] = True
            for x, pool, scales in ((key, after.key, after.key_scale), (value, after.value, after.value_scale)):
                x = x[b, t].cpu()
                if not scaled:
                    assert torch.equal(_bits(pool[page, slot].cpu().contiguous()), _bits(x.contiguous()))
                    continue
                want, s = ref.quantise(x)
                got_s = scales[page, slot].cpu().double()
                assert ((got_s - s).abs() <= 2.0 ** -24 * s).all()
                # half an e4m3 step (the smallest: 2**-9), and the 32-bit factor before the rounding
                got = pool[page, slot].cpu().double()
                tol = torch.clamp_min(want.abs() * 2.0 ** -4, 2.0 ** -10) + 2.0 ** -22 * want.abs()
                assert ((got - want).abs() <= tol).all()
    for x, y in zip(before, after):
        if x is not None:
            keep = ~touched.cuda()
            assert torch.equal(_bits(x)[keep], _bits(y)[keep])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("eight_bits", [False, True])
@pytest.mark.parametrize("batch,tokens,heads,dim,page", [
    (1, 1, 1, 1, 1), (3, 1, 2, 64, 16), (2, 37, 3, 80, 20), (2, 5, 4, 128, 64), (1, 300, 2, 33, 7),
    (2, 9, 1, 256, 8), (4, 3, 2, 255, 16), (2, 70, 8, 48, 32)])
def test_write_and_read_back(dtype, eight_bits, batch, tokens, heads, dim, page):
    torch.manual_seed(1)
    per = -(-(tokens + 2 * page) // page)
    pages = batch * per + 2
    cache = _filled(pages, page, heads, dim, E4M3 if eight_bits else dtype)
    table = torch.randperm(pages, device="cuda")[:batch * per].view(batch, per).int()
    start = torch.randint(0, page + 1, (batch,), device="cuda", dtype=torch.int32)
    counts = torch.randint(0, tokens + 1, (batch,), device="cuda", dtype=torch.int32)
    counts[0] = tokens
    kv = torch.randn(batch, tokens, heads, 2, dim, device="cuda") * torch.exp(torch.randn(dim, device="cuda"))
    key, value = kv.to(dtype).unbind(3)                    # strided
    before = _clone(cache)
    nb.kv_cache_write(cache, key, value, table, start, counts)
    _check_write(before, cache, key, value, table, start, counts)

    length = tokens + 3
    got = nb.kv_cache_read(cache, table, length, start, counts, dtype=dtype)
    for g, pool, scales in zip(got, cache[:2], (cache.key_scale, cache.value_scale)):
        assert g.shape == (batch, length, heads, dim) and g.dtype == dtype and g.is_contiguous()
        for b in range(batch):
            n = int(counts[b])
            rows, ok = ref.cached_rows(pool.cpu(), None if scales is None else scales.cpu(), table[b].cpu(),
                                       range(int(start[b]), int(start[b]) + n))
            assert ok.all()
            # one 32-bit product and its rounding to the type; nothing is rounded without a scale
            tol = rows.abs() * (ref.HALF_STEP[dtype] + 2.0 ** -24) + 2.0 ** -25 if eight_bits else 0 * rows
            ref.assert_close(g[b, :n], rows, tol)
            assert not g[b, n:].any()


@pytest.mark.parametrize("eight_bits", [False, True])
def test_places_that_are_no_page(eight_bits):
    torch.manual_seed(2)
    cache = _filled(5, 4, 2, 16, E4M3 if eight_bits else torch.bfloat16)
    table = torch.tensor([[-1, 0, 5], [2 ** 31 - 1, -2 ** 31, 1], [3, 4, 2]], dtype=torch.int32, device="cuda")
    start = torch.tensor([-2, 1, 7], dtype=torch.int32, device="cuda")
    counts = torch.tensor([100, -3, 14], dtype=torch.int32, device="cuda")
    x = torch.randn(3, 14, 2, 16, device="cuda").bfloat16()
    before = _clone(cache)
    nb.kv_cache_write(cache, x, -x, table, start, counts)
    _check_write(before, cache, x, -x, table, start, counts)
    key, value = nb.kv_cache_read(cache, table, 14, start, counts)
    for b in range(3):
        for t in range(14):
            p = int(start[b]) + t
            page = int(table[b, p // 4]) if p >= 0 and p // 4 < 3 else -1
            on = t < int(counts[b]) and 0 <= page < 5
            assert bool(key[b, t].any()) == on and bool(value[b, t].any()) == on
    # no pages at all, no columns, no tokens
    empty = nb.KVCache.allocate(0, 4, 2, 16)
    nb.kv_cache_write(empty, x, x, table)
    assert not nb.kv_cache_read(empty, table, 3)[0].any()
    assert nb.kv_cache_read(cache, table, 0)[0].shape == (3, 0, 2, 16)
    nb.kv_cache_write(cache, x[:, :0], x[:, :0], table)
    nb.kv_cache_write(cache, x[:0], x[:0], table[:0])
    none = table[:, :0]
    nb.kv_cache_write(cache, x, x, none)
    assert not nb.kv_cache_read(cache, none, 3, dtype=torch.bfloat16)[0].any()


@pytest.mark.parametrize("dtype", DTYPES)
def test_rows_of_every_kind_in_eight_bits(dtype):
    """Zeros, the smallest and largest magnitudes, not-a-numbers: a row that is not finite reads back as
    NaN, its neighbours do not."""
    info = torch.finfo(dtype)
    rows = torch.zeros(8, 32, dtype=torch.float64)
    rows[1, 3] = info.tiny
    rows[2] = torch.linspace(-1, 1, 32, dtype=torch.float64) * info.max
    rows[3, 0], rows[3, 1] = info.max, info.tiny
    rows[4] = torch.randn(32).double()
    rows[5, 9] = math.nan
    rows[6, 9] = math.inf
    rows[7] = -torch.randn(32).double() * (1e-6 if dtype == torch.float16 else 1e-36)
    x = rows.to(dtype).view(1, 8, 1, 32).cuda()
    cache = nb.KVCache.allocate(2, 4, 1, 32, E4M3)
    table = torch.tensor([[1, 0]], dtype=torch.int32, device="cuda")
    nb.kv_cache_write(cache, x, x, table)
    got = nb.kv_cache_read(cache, table, 8, dtype=torch.float32)[0].cpu().double()[0, :, 0]
    assert torch.isnan(got[5]).all() and torch.isnan(got[6]).all()
    fine = [0, 1, 2, 3, 4, 7]
    want = x.cpu().double()[0, :, 0][fine]
    q, s = ref.quantise(want)
    tol = torch.clamp_min(q.abs() * (2.0 ** -4 + 2.0 ** -20), 2.0 ** -10) * s[:, None]
    assert ((got[fine] - want).abs() <= tol).all()
    assert not got[0].any()


def test_pools_in_other_strides():
    torch.manual_seed(3)
    for dtype in (torch.bfloat16, E4M3):
        plain = _filled(6, 8, 3, 64, dtype)
        # heads before slots; every other page of a larger pool; keys and values of one pool, off 16 bytes
        heads_first = nb.KVCache(*(None if t is None else t.transpose(1, 2).contiguous().transpose(1, 2)
                                   for t in plain))
        both = torch.zeros(6, 8, 3, 2, 65, device="cuda").to(dtype)
        shifted = nb.KVCache(both[..., 0, 1:], both[..., 1, :64])
        if dtype == E4M3:
            s = torch.zeros(12, 8, 3, 2, device="cuda")
            shifted = nb.KVCache(both[..., 0, 1:], both[..., 1, :64], s[::2, ..., 0], s[::2, ..., 1])
        table = torch.tensor([[3, 0], [5, 1]], dtype=torch.int32, device="cuda")
        wide = torch.full((2, 6), -1, dtype=torch.int32, device="cuda")
        wide[:, ::3] = table
        x = torch.randn(2, 13, 3, 64, device="cuda").bfloat16()
        y = torch.randn(2, 13, 3, 64, device="cuda").bfloat16()
        want = None
        for c in (plain, heads_first, shifted):
            for tab in (table, wide[:, ::3], table.t().contiguous().t()):
                nb.kv_cache_write(c, x, y, tab)
                got = nb.kv_cache_read(c, tab, 16, counts=torch.tensor([13, 12], dtype=torch.int32,
                                                                       device="cuda"))
                want = want or got
                assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_rows_beyond_32_bit_offsets():
    """The last page of a pool of more than 2^31 elements."""
    pages, page, heads, dim = 2 ** 16 + 2, 64, 4, 128
    pool = torch.zeros(pages, page, heads, dim, dtype=torch.bfloat16, device="cuda")
    cache = nb.KVCache(pool, pool)
    table = torch.tensor([[pages - 1, 0]], dtype=torch.int32, device="cuda")
    x = torch.randn(1, 70, heads, dim, device="cuda").bfloat16()
    nb.kv_cache_write(cache, x, x, table)
    assert torch.equal(pool[-1], x[0, :64]) and torch.equal(pool[0, :6], x[0, 64:])
    assert torch.equal(nb.kv_cache_read(cache, table, 70)[1], x)
    q = torch.randn(1, 1, 4, dim, device="cuda").bfloat16()
    n = torch.tensor([70], dtype=torch.int32, device="cuda")
    out, lse = nb.na1d_decode(q, cache, table, n, return_lse=True)
    want = ref.decode(q.cpu(), (x.cpu(), x.cpu(), None, None), torch.zeros(1, 1, dtype=torch.int32), [70], 0,
                      1, dim ** -0.5, 2.0 ** -8)     # one page that holds all of it
    ref.assert_close(out, want[0], want[2])
    ref.assert_close(lse, want[1], want[3])


def test_other_stream_captured_and_compiled():
    torch.manual_seed(4)
    cache = _filled(8, 8, 2, 32, E4M3)
    table = torch.randperm(8, device="cuda").view(2, 4).int()
    x = torch.randn(2, 20, 2, 32, device="cuda").bfloat16()
    start = torch.tensor([3, 0], dtype=torch.int32, device="cuda")
    counts = torch.tensor([20, 11], dtype=torch.int32, device="cuda")
    for c in (cache, _filled(8, 8, 2, 32, torch.bfloat16)):
        # (the schema check multiplies what it is given, which torch does not do in 8 bits)
        tests = ("test_faketensor",) if c is cache else ("test_schema", "test_faketensor")
        torch.library.opcheck(ops.kv_cache_write, (x, x, *c, table, start, counts), test_utils=tests)
        torch.library.opcheck(ops.kv_cache_read, (*c, table, start, counts, 20, torch.bfloat16),
                              test_utils=tests)

    def f(x, start):
        nb.kv_cache_write(cache, x * 2.0, x, table, start, counts)
        return nb.kv_cache_read(cache, table, 23, dtype=torch.float32)

    want = f(x, start)
    got = torch.compile(f, fullgraph=True)(x, start)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = f(x, start)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got[0], want[0])
    s = start.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = f(x, s)
    for v in ((3, 0), (1, 9)):
        s.copy_(torch.tensor(v, dtype=torch.int32))
        graph.replay()
        mine = [t.clone() for t in got]
        again = f(x, s)
        assert torch.equal(mine[0], again[0]) and torch.equal(mine[1], again[1])
