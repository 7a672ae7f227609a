"""Attention of the newest tokens over a paged cache against a plain 64-bit form."""
import math

import pytest
import torch

import natten_b200 as nb
import natten_b200._lib as L
import serving_reference as ref
from natten_b200 import ops

pytestmark = pytest.mark.gpu
E4M3 = torch.float8_e4m3fn


def _state(dtype, cache_dtype, lengths, tokens, heads, heads_kv, dim, page, spread=1.0, seed=0):
    torch.manual_seed(seed)
    per = max(1, max(-(-max(n, 1) // page) for n in lengths))
    pages = len(lengths) * per + 1
    cache = nb.KVCache.allocate(pages, page, heads_kv, dim, cache_dtype)
    # what was never written must not be read: not-a-numbers everywhere first
    for t in cache:
        if t is not None:
            t.copy_(torch.full(t.shape, math.nan, device="cuda").to(t.dtype))
    table = torch.randperm(pages, device="cuda")[:len(lengths) * per].view(len(lengths), per).int()
    n = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    kv_dtype = dtype
    longest = max(max(lengths), 1)
    key, value = (torch.randn(len(lengths), longest, heads_kv, dim, device="cuda").to(kv_dtype)
                  for _ in range(2))
    nb.kv_cache_write(cache, key, value + 0.5, table, counts=n)
    query = (spread * torch.randn(len(lengths), tokens, heads, dim, device="cuda")).to(dtype)
    return query, cache, table, n


def _weight_step(dtype, cache_dtype):
    if dtype == torch.float32:
        return 2.0 ** -24
    return 2.0 ** -11 if cache_dtype == E4M3 else ref.HALF_STEP[dtype]


def _check(query, cache, table, lengths, kernel_size=None, dilation=1, scale=None):
    out, lse = nb.na1d_decode(query, cache, table, lengths, kernel_size, dilation, scale, return_lse=True)
    assert out.shape == query.shape and out.dtype == query.dtype and out.is_contiguous()
    assert lse.shape == query.shape[:-1] and lse.dtype == torch.float32
    cpu = nb.KVCache(*(None if t is None else t.cpu() for t in cache))
    want, want_lse, tol, tol_lse = ref.decode(query.cpu(), cpu, table.cpu(), lengths.tolist(), kernel_size or 0,
                                              dilation, scale or query.shape[-1] ** -0.5,
                                              _weight_step(query.dtype, cache.key.dtype))
    ref.assert_close(out, want, tol)
    ref.assert_close(lse, want_lse, tol_lse)
    return out, lse


TYPES = [(torch.float32, torch.float32), (torch.float16, torch.float16), (torch.bfloat16, torch.bfloat16),
         (torch.float32, E4M3), (torch.float16, E4M3), (torch.bfloat16, E4M3)]


@pytest.mark.parametrize("dtype,cache_dtype", TYPES)
@pytest.mark.parametrize("lengths,tokens,heads,heads_kv,dim,page,kernel_size,dilation", [
    ([1], 1, 1, 1, 64, 16, None, 1),
    ([0, 1, 2, 15, 16, 17, 63, 64, 65, 129], 1, 4, 2, 64, 16, None, 1),       # lengths of zero and one
    ([300, 5, 77], 1, 8, 1, 128, 20, 64, 1),                                  # pages end inside a tile
    ([500, 333], 1, 7, 7, 128, 64, 100, 1),                                   # a head of its own each
    ([700, 41], 1, 6, 2, 48, 7, 50, 5),                                       # dilated
    ([700, 41, 3], 4, 6, 2, 80, 32, 33, 3),                                   # dilated, drafted tokens
    ([200, 3, 0, 64], 5, 12, 4, 64, 16, 40, 1),                               # fewer tokens than queries
    ([130, 70], 9, 8, 2, 128, 16, None, 1),
    ([90, 200], 3, 34, 2, 64, 64, None, 1),                                   # 17 heads a group
    ([257], 1, 80, 1, 64, 16, 200, 1),                                        # 80 heads a group
    ([150, 31], 2, 4, 2, 256, 16, None, 1),
    ([150, 31], 1, 4, 2, 16, 16, None, 1),
    ([150, 31], 2, 2, 2, 208, 16, 90, 1),
    ([64, 31], 17, 2, 2, 32, 8, 20, 1),                                       # more queries than a window
    ([70, 12], 2, 4, 4, 64, 1, 30, 1),                                        # pages of one token
    ([300], 1, 4, 2, 128, 1024, None, 2),                                     # one page, dilated, all of it
])
def test_shapes(dtype, cache_dtype, lengths, tokens, heads, heads_kv, dim, page, kernel_size, dilation):
    _check(*_state(dtype, cache_dtype, lengths, tokens, heads, heads_kv, dim, page), kernel_size, dilation)


@pytest.mark.parametrize("dtype,cache_dtype", TYPES)
@pytest.mark.parametrize("dim", [1, 7, 33, 72, 100, 255])
def test_odd_heads(dtype, cache_dtype, dim):
    _check(*_state(dtype, cache_dtype, [77, 140], 2, 4, 2, dim, 16), 100)


@pytest.mark.parametrize("dtype,cache_dtype", TYPES)
def test_long_ragged_batches(dtype, cache_dtype):
    """Sequences over many blocks next to sequences that share one; more sequences than threads."""
    _check(*_state(dtype, cache_dtype, [9000, 3, 0, 64, 2500, 1], 1, 4, 1, 64, 64))
    lengths = [(37 * i) % 150 for i in range(300)]
    _check(*_state(dtype, cache_dtype, lengths, 1, 2, 1, 32, 16), 40)


@pytest.mark.parametrize("dtype,cache_dtype", TYPES)
def test_peaked_and_flat_rows(dtype, cache_dtype):
    _check(*_state(dtype, cache_dtype, [600, 90], 2, 4, 2, 64, 16, spread=12.0))
    _check(*_state(dtype, cache_dtype, [600, 90], 2, 4, 2, 64, 16, spread=0.0))
    _check(*_state(dtype, cache_dtype, [600, 90], 2, 4, 2, 64, 16), scale=1e-3)
    _check(*_state(dtype, cache_dtype, [600, 90], 2, 4, 2, 64, 16, spread=1e-6), scale=1e5)


def test_eight_bit_rows_of_very_different_size():
    """Values whose scales lie far apart: a row that attends the small ones alone keeps their precision."""
    q, cache, table, n = _state(torch.float16, E4M3, [40], 1, 2, 2, 64, 8)
    key = torch.randn(1, 40, 2, 64, device="cuda").half()
    key[0, 10] = 8 * q[0, 0]                              # all of the weight
    value = torch.randn(1, 40, 2, 64, device="cuda").half()
    value[0, 10] *= 2.0 ** -12
    value[0, 11] *= 2.0 ** 13
    nb.kv_cache_write(cache, key, value, table)
    _check(q, cache, table, n, scale=1.0)
    _check(q, cache, table, n, scale=1e-3)


def test_queries_and_pools_in_other_strides():
    for dtype, cache_dtype in ((torch.bfloat16, torch.bfloat16), (torch.bfloat16, E4M3),
                               (torch.float32, torch.float32)):
        q, cache, table, n = _state(dtype, cache_dtype, [100, 61], 3, 8, 2, 64, 16)
        want, _ = _check(q, cache, table, n, 70)
        heads_first = nb.KVCache(*(None if t is None else t.transpose(1, 2).contiguous().transpose(1, 2)
                                   for t in cache))
        fused = torch.randn(2, 3, 12, 64, device="cuda").to(dtype)
        fused[:, :, 2:10] = q
        flat = torch.zeros(q.numel() + 1, device="cuda", dtype=dtype)
        flat[1:] = q.flatten()
        wide = torch.full((2, 2 * table.shape[1]), 0, dtype=torch.int32, device="cuda")
        wide[:, ::2] = table
        for c in (cache, heads_first):
            for x in (fused[:, :, 2:10], flat[1:].view_as(q), q.transpose(1, 2).contiguous().transpose(1, 2),
                      q.transpose(-1, -2).contiguous().transpose(-1, -2)):
                assert torch.equal(nb.na1d_decode(x, c, wide[:, ::2], n, 70), want)
        # pools off 16-byte boundaries, keys and values in strides of their own
        big = torch.zeros(*cache.key.shape[:3], 2, 65, device="cuda").to(cache_dtype)
        big[..., 0, 1:], big[..., 1, :64] = cache.key, cache.value
        _check(q, nb.KVCache(big[..., 0, 1:], big[..., 1, :64], *cache[2:]), table, n, 70)


@pytest.mark.parametrize("dtype,cache_dtype", TYPES)
@pytest.mark.parametrize("tokens,heads", [(1, 2), (4, 8), (6, 2)])
def test_non_finite_values_stay_with_the_rows_that_attend_them(dtype, cache_dtype, tokens, heads):
    for where in ("key", "value"):
        for bad in (math.nan, math.inf, -math.inf):
            q, cache, table, n = _state(dtype, cache_dtype, [90, 90], tokens, heads, 2, 64, 16, seed=3)
            pool = getattr(cache, where)
            # in the newest token of sequence 0; just before its window; far behind the cached tokens
            for b, p in ((0, 89), (0, 89 - 40 - tokens + 1)):
                page = table[b, p // 16]
                if cache_dtype == E4M3:
                    getattr(cache, where + "_scale")[page, p % 16] = bad
                else:
                    pool[page, p % 16, 0, 5] = bad
            out, lse = nb.na1d_decode(q, cache, table, n, 40, return_lse=True)
            per = heads // 2
            hit = torch.zeros(2, tokens, heads, dtype=torch.bool, device="cuda")
            last = slice(0, heads) if cache_dtype == E4M3 else slice(0, per)
            hit[0, -1, last] = True
            assert torch.isfinite(out[~hit]).all() and torch.isfinite(lse[~hit]).all()
            clean = _state(dtype, cache_dtype, [90, 90], tokens, heads, 2, 64, 16, seed=3)
            good = nb.na1d_decode(*clean, 40)
            assert torch.equal(out[~hit], good[~hit])
            if where == "value":
                assert not torch.isfinite(out[hit]).all(-1).any()
            elif math.isnan(bad):
                assert torch.isnan(out[hit]).all() and torch.isnan(lse[hit]).all()


def test_no_page_and_tables_shorter_than_the_lengths():
    for dtype, cache_dtype in ((torch.bfloat16, torch.bfloat16), (torch.float32, torch.float32),
                               (torch.float16, E4M3)):
        q, cache, table, n = _state(dtype, cache_dtype, [100, 100, 100, 40], 2, 4, 2, 64, 16)
        table[0, 1], table[0, 3] = -1, 10 ** 6          # holes
        table[1] = -1                                   # nothing there
        table[2, -1] = 2 ** 31 - 1                      # the newest tokens are not there
        _check(q, cache, table, n)
        _check(q, cache, table, n, 30)
        _check(q, cache, table, n, 9, 7)
        # lengths that a table cannot name, and negative ones
        odd = torch.tensor([2 ** 31 - 1, -5, 120, 99], dtype=torch.int32, device="cuda")
        out, lse = nb.na1d_decode(q, cache, table, odd, 64, return_lse=True)
        assert not out[:2].any() and torch.isneginf(lse[:2]).all()
        assert torch.isfinite(out[2]).all()     # (the last one attends what was never written)
        _check(q[2:], cache, table[2:], odd[2:], 64)
        # pages behind the window given back: the same bits
        q, cache, table, n = _state(dtype, cache_dtype, [100, 77], 1, 4, 2, 64, 16)
        want = nb.na1d_decode(q, cache, table, n, 20)
        table[0, :5] = -1
        assert torch.equal(nb.na1d_decode(q, cache, table, n, 20), want)
        none = nb.KVCache.allocate(0, 16, 2, 64, cache_dtype)
        assert not nb.na1d_decode(q, none, table, n).any()
        assert not nb.na1d_decode(q, cache, table[:, :0], n).any()
        assert nb.na1d_decode(q[:0], cache, table[:0], n[:0]).shape == (0, 1, 4, 64)
        assert nb.na1d_decode(q[:, :0], cache, table, n).shape == (2, 0, 4, 64)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("kernel_size,dilation", [(64, 1), (33, 3), (300, 1)])
def test_last_rows_of_na1d(dtype, kernel_size, dilation):
    """The same rows that the training and prefill operator gives (stride 1, causal)."""
    torch.manual_seed(5)
    q, k, v = (torch.randn(2, 300, h, 64, device="cuda").to(dtype) for h in (4, 2, 2))
    full, full_lse = nb.na1d(q, k, v, kernel_size, 1, dilation, True, return_lse=True)
    cache = nb.KVCache.allocate(40, 16, 2, 64, dtype)
    table = torch.randperm(40, device="cuda")[:38].view(2, 19).int()
    nb.kv_cache_write(cache, k, v, table)
    for end, tokens in ((300, 1), (300, 7), (1, 1), (150, 150)):
        n = torch.full((2,), end, dtype=torch.int32, device="cuda")
        out, lse = nb.na1d_decode(q[:, end - tokens:end], cache, table, n, kernel_size, dilation,
                                  return_lse=True)
        # both round their weights and results to the type: two half steps of each, values of 5 at most
        tol = 4 * ref.HALF_STEP[dtype] * 5
        assert (out.float() - full[:, end - tokens:end].float()).abs().max() <= tol
        assert (lse - full_lse[:, end - tokens:end]).abs().max() <= 1e-3


def test_merges_with_attention_over_other_tokens():
    q, cache, table, n = _state(torch.bfloat16, torch.bfloat16, [120, 64], 1, 4, 4, 64, 16)
    k, v = (torch.randn(2, 50, 4, 64, device="cuda").bfloat16() for _ in range(2))
    a, la = nb.na1d_decode(q, cache, table, n, return_lse=True)
    b, lb = nb.attention(q, k, v, return_lse=True)
    out, lse = nb.merge_attentions([a, b], [la, lb])
    for i in range(2):
        m = int(n[i])
        kk, vv = nb.kv_cache_read(cache, table[i:i + 1], m)
        want, want_lse = nb.attention(q[i:i + 1], torch.cat((kk, k[i:i + 1]), 1), torch.cat((vv, v[i:i + 1]), 1),
                                      return_lse=True)
        assert (out[i:i + 1].float() - want.float()).abs().max() <= 4 * 2.0 ** -8 * 5
        assert (lse[i:i + 1] - want_lse).abs().max() <= 1e-3


def test_same_bits_every_time_and_on_every_stream():
    states = [_state(torch.bfloat16, c, [5000, 31, 800], 1, 8, 2, 128, 64, seed=s)
              for s, c in enumerate((torch.bfloat16, E4M3, torch.bfloat16))]
    want = [nb.na1d_decode(*s, return_lse=True) for s in states]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in states]
    for _ in range(5):
        got = []
        for st, s in zip(streams, states):
            with torch.cuda.stream(st):
                got.append(nb.na1d_decode(*s, return_lse=True))
        torch.cuda.synchronize()
        for g, w in zip(got, want):
            assert torch.equal(g[0], w[0]) and torch.equal(g[1], w[1])


def test_captured_steps_follow_lengths_and_tables():
    q, cache, table, n = _state(torch.bfloat16, torch.bfloat16, [300, 300, 300], 2, 8, 2, 64, 16)
    graphs, outs = [], []
    tables, lengths = [table.clone() for _ in range(2)], [n.clone() for _ in range(2)]
    for i in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(nb.na1d_decode(q, cache, tables[i], lengths[i], 200, return_lse=True))
        graphs.append(g)
    for step in ([300, 1, 0], [7, 299, 64], [128, 128, 300]):
        for i in range(2):
            lengths[i].copy_(torch.tensor(step[i:] + step[:i], dtype=torch.int32))
            tables[i].copy_(table.roll(i + 1, 0))
        streams = [torch.cuda.Stream() for _ in range(2)]
        torch.cuda.synchronize()
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for i in range(2):
            want = nb.na1d_decode(q, cache, tables[i], lengths[i], 200, return_lse=True)
            assert torch.equal(outs[i][0], want[0]) and torch.equal(outs[i][1], want[1])


def test_op_and_compile():
    q, cache, table, n = _state(torch.bfloat16, E4M3, [100, 61], 1, 8, 2, 64, 16)
    torch.library.opcheck(ops.na1d_decode, (q, *cache, table, n, 40, 1, 0.125),
                          test_utils=("test_faketensor",))
    half = _state(torch.bfloat16, torch.bfloat16, [100, 61], 1, 8, 2, 64, 16)
    torch.library.opcheck(ops.na1d_decode, (torch.zeros_like(q), *(None if t is None else torch.zeros_like(t)
                                                                   for t in half[1]), table, n, 40, 1, 0.125),
                          test_utils=("test_schema", "test_faketensor"))

    def f(q):
        out, lse = nb.na1d_decode(q * 2.0, cache, table, n, 40, return_lse=True)
        return out.float() + 1.0, lse

    want, got = f(q), torch.compile(f, fullgraph=True)(q)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    assert L.device_status() == 0


@pytest.mark.parametrize("cache_dtype", [torch.bfloat16, E4M3])
def test_a_run_of_them_together(cache_dtype):
    """Prompt and steps of a causal model: rotary positions, the cache written, attention over it, against
    the same model without a cache."""
    torch.manual_seed(9)
    B, N, heads, heads_kv, dim, prompt = 2, 90, 4, 2, 64, 70
    q, k, v = (torch.randn(B, N, h, dim, device="cuda").bfloat16() for h in (heads, heads_kv, heads_kv))
    qr, kr = nb.rotary(q, k)
    want = nb.na1d(qr, kr, v, 32, is_causal=True)
    cache = nb.KVCache.allocate(30, 8, heads_kv, dim, cache_dtype)
    table = torch.randperm(30, device="cuda")[:24].view(B, 12).int()
    nb.kv_cache_write(cache, kr[:, :prompt], v[:, :prompt], table)
    # 8 bits: half a step of every value (relative to a row's largest, about 3) and of every logit
    tol = 4 * 2.0 ** -8 * 5 + (2.0 ** -4 * 4 if cache_dtype == E4M3 else 0)
    at = prompt
    for tokens in (1, 1, 4, 1, 8, 1, 4):
        start = torch.full((B,), at, dtype=torch.int32, device="cuda")
        positions = (start[:, None] + torch.arange(tokens, device="cuda", dtype=torch.int32))[..., None]
        qs, ks = nb.rotary(q[:, at:at + tokens], k[:, at:at + tokens], positions=positions)
        assert torch.equal(ks, kr[:, at:at + tokens])
        nb.kv_cache_write(cache, ks, v[:, at:at + tokens], table, start)
        out = nb.na1d_decode(qs, cache, table, start + tokens, 32)
        assert (out.float() - want[:, at:at + tokens].float()).abs().max() <= tol
        at += tokens
    assert at == N
    key, value = nb.kv_cache_read(cache, table, N)
    if cache_dtype == torch.bfloat16:
        assert torch.equal(key, kr) and torch.equal(value, v)


def test_native_front_and_registered_operators_give_the_same(monkeypatch):
    """The call from C++ and the one through the registered operators, and the versions of what they
    write."""
    import natten_b200.kv_cache as module
    for dtype, cache_dtype in TYPES:
        q, cache, table, n = _state(dtype, cache_dtype, [120, 64], 3, 4, 2, 64, 16)
        k = torch.randn(2, 3, 2, 64, device="cuda").to(dtype)
        got = []
        for native in (True, False):
            monkeypatch.setattr(module, "_native_eligible", lambda native=native: native)
            c = nb.KVCache(*(None if t is None else t.clone() for t in cache))
            version = c.key._version
            nb.kv_cache_write(c, k, k, table, n - 3, counts=torch.full_like(n, 2))
            assert c.key._version > version
            got.append((*c[:2], *nb.kv_cache_read(c, table, 130, dtype=dtype),
                        *nb.na1d_decode(q, c, table, n, 50, return_lse=True), nb.na1d_decode(q, c, table, n)))
        for x, y in zip(*got):
            assert torch.equal(x.view(torch.uint8), y.view(torch.uint8))
    before = L.launches
    monkeypatch.setattr(module, "_native_eligible", lambda: True)
    nb.na1d_decode(q, c, table, n)
    nb.kv_cache_read(c, table, 5, dtype=dtype)
    assert L.launches == before + 2      # (a short table: one launch each)
    before = L.launches
    nb.na1d_decode(q, c, table.repeat(1, 3000), n)
    assert L.launches == before + 2      # ranges of all sequences' keys, and their join


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("tokens,heads", [(1, 2), (1, 24), (4, 8)])
def test_an_8_bit_element_that_is_no_number(dtype, tokens, heads):
    """A NaN in the pool itself: of a key it reaches the rows that attend it, of a value their channel."""
    for where in ("key", "value"):
        q, cache, table, n = _state(dtype, E4M3, [90, 90], tokens, heads, 2, 64, 16, seed=4)
        good = nb.na1d_decode(q, cache, table, n, 40)
        pool = getattr(cache, where)
        for p in (89, 89 - 40 - tokens + 1):        # the newest token; the last one before all windows
            pool.view(torch.uint8)[table[0, p // 16].long(), p % 16, 0, 5] = 0x7F
        out, lse = nb.na1d_decode(q, cache, table, n, 40, return_lse=True)
        hit = torch.zeros(2, tokens, heads, 64, dtype=torch.bool, device="cuda")
        hit[0, -1, :heads // 2, slice(None) if where == "key" else 5] = True
        assert torch.isnan(out[hit]).all() and torch.equal(out[~hit], good[~hit])
        assert torch.equal(torch.isnan(lse), hit.all(-1))


def test_many_rows_and_ranges_of_wide_heads():
    """Items of 16 rows over ranges and their join; heads that fill an SM's shared memory."""
    for dtype, cache_dtype in TYPES:
        _check(*_state(dtype, cache_dtype, [12000, 40], 1, 16, 1, 128, 64))
        _check(*_state(dtype, cache_dtype, [9000, 500, 1], 3, 4, 1, 256, 64))


FIRST_CALLS = """
import torch
import natten_b200 as nb
torch.zeros(1, device="cuda")
cache = nb.KVCache.allocate(8, 16, 2, 64, torch.float8_e4m3fn)
table = torch.arange(8, device="cuda").int().view(1, 8)
n = torch.full((1,), 100, dtype=torch.int32, device="cuda")
q, k = torch.randn(1, 100, 4, 64, device="cuda").bfloat16(), torch.randn(1, 100, 2, 64, device="cuda").bfloat16()
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    a, b = nb.rotary(q, k)
    nb.kv_cache_write(cache, b, b, table)
    key, value = nb.kv_cache_read(cache, table, 100)
    outs = [nb.na1d_decode(a[:, -t:], cache, table, n, w) for t in (1, 8) for w in (None, 40)]
graph.replay()
torch.cuda.synchronize()
mine = [t.clone() for t in (a, b, key, value, *outs)]
a, b = nb.rotary(q, k)
nb.kv_cache_write(cache, b, b, table)
again = [a, b, *nb.kv_cache_read(cache, table, 100)]
again += [nb.na1d_decode(a[:, -t:], cache, table, n, w) for t in (1, 8) for w in (None, 40)]
assert all(torch.equal(x, y) for x, y in zip(mine, again))
print("the same")
"""


def test_first_calls_of_a_process_may_be_captured():
    """These kernels need no set-up of the device before they are recorded."""
    import os
    import subprocess
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    done = subprocess.run([sys.executable, "-c", FIRST_CALLS], cwd=root, capture_output=True, text=True, timeout=300)
    assert done.returncode == 0 and "the same" in done.stdout, done.stdout + done.stderr
