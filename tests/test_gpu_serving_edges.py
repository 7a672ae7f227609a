"""The serving operators at the edges of what they accept, on the GPU: each test holds a call that once gave
something else than its definition."""
import math

import pytest
import torch

import natten_b200 as nb
import serving_reference as ref
from test_gpu_decode import E4M3, TYPES, _check, _state

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,cache_dtype", TYPES)
@pytest.mark.parametrize("heads", [4, 24])
def test_an_infinite_query_that_attends_nothing(dtype, cache_dtype, heads):
    """Zeros and -inf like any other row without tokens (a drafted place that a short sequence does not
    have, a table without pages); where there are tokens, the row alone is not finite."""
    q, cache, table, n = _state(dtype, cache_dtype, [1, 40, 40], 2, heads, 2, 64, 16)
    table[1] = -1
    for kernel_size in (None, 30):
        good, good_lse = nb.na1d_decode(q, cache, table, n, kernel_size, return_lse=True)
        bad = q.clone()
        bad[0, 0, :, 3] = math.inf
        bad[1, :, :, 5] = -math.inf
        bad[2, 0, 0, 7] = math.inf
        out, lse = nb.na1d_decode(bad, cache, table, n, kernel_size, return_lse=True)
        for rows in ((0, 0), (1, 0), (1, 1)):
            assert not out[rows].any() and torch.isneginf(lse[rows]).all()
        assert torch.isnan(out[2, 0, 0]).all()
        out[2, 0, 0], lse[2, 0, 0] = good[2, 0, 0], good_lse[2, 0, 0]
        assert torch.equal(out, good) and torch.equal(lse, good_lse)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_eight_bit_rows_are_divided_by_their_scale(dtype):
    """The bytes of x / scale (one 32-bit division, one rounding to e4m3) and max|x| / 448, for rows with every
    largest mantissa of bf16 (128 of them) next to every bf16 value of the ten octaves below, in which values
    half-way between two e4m3 numbers occur; at the smallest and largest magnitudes of the type, too."""
    torch.manual_seed(1)
    mantissas = 1 + torch.arange(128) / 128
    values = torch.cat([mantissas * 2.0 ** -e for e in range(10)])            # 1280
    rows = torch.zeros(128, 6, 256)
    for i in range(6):
        some = values[214 * i:214 * (i + 1)]
        rows[:, i, 1:1 + len(some)] = torch.minimum(some, mantissas[:, None])
        rows[:, i, 0] = mantissas
    rows = (rows * torch.where(torch.rand(rows.shape) < 0.5, -1.0, 1.0)).flatten(0, 1)
    ups = [1.0, 2.0 ** -10, 2.0 ** 14] if dtype == torch.float16 else [1.0, 2.0 ** -125, 2.0 ** -117, 2.0 ** -60,
                                                                       2.0 ** 100, 2.0 ** 126]
    x = torch.cat([rows * up for up in ups]).to(dtype)
    tokens = x.shape[0]
    for dim in (256, 255):                                                     # rows in wide accesses, and not
        part = x[:, :dim].reshape(1, tokens, 1, dim)
        cache = nb.KVCache.allocate(-(-tokens // 64), 64, 1, dim, E4M3)
        table = torch.arange(cache.key.shape[0], dtype=torch.int32, device="cuda").view(1, -1)
        nb.kv_cache_write(cache, part.cuda(), -part.cuda(), table)
        full = part[0, :, 0].float()
        scale = torch.clamp_min(full.abs().amax(-1) / 448.0, 2.0 ** -126)
        for pool, scales, sign in ((cache.key, cache.key_scale, 1.0), (cache.value, cache.value_scale, -1.0)):
            assert torch.equal(scales.flatten()[:tokens].cpu(), scale)
            want = (sign * full / scale[:, None]).to(E4M3)
            got = pool.view(-1, dim)[:tokens].cpu()
            assert torch.equal(got.view(torch.uint8), want.view(torch.uint8))


@pytest.mark.parametrize("dtype,cache_dtype", [t for t in TYPES if t[0] != torch.float16])
@pytest.mark.parametrize("heads", [4, 24])
def test_logits_smaller_than_32_bits_hold(dtype, cache_dtype, heads):
    """Queries of 2**-100 with a scale of 2**-60: every logit is nothing, every token that is there weighs
    the same, and holes weigh nothing."""
    q, cache, table, n = _state(dtype, cache_dtype, [90, 33], 2, heads, 2, 64, 16, spread=2.0 ** -100)
    table[0, 1] = -1
    _check(q, cache, table, n, scale=2.0 ** -60)
    _check(q, cache, table, n, 20, scale=2.0 ** -60)


@pytest.mark.parametrize("heads", [4, 24])
def test_queries_near_the_largest_number(heads):
    """bf16 queries of 2**127 and more on keys of about 2**-125."""
    q, cache, table, n = _state(torch.bfloat16, E4M3, [90, 33], 2, heads, 2, 64, 16)
    big = torch.finfo(torch.bfloat16).max
    q = ((torch.rand(q.shape, device="cuda") * 0.5 + 0.5) * torch.sign(q.float()) * big).bfloat16()
    key = (torch.randn(2, 90, 2, 64, device="cuda") * 2.0 ** -125).bfloat16()
    value = torch.randn(2, 90, 2, 64, device="cuda").bfloat16()
    nb.kv_cache_write(cache, key, value, table, counts=n)
    _check(q, cache, table, n)


def test_rotary_turns_keys_beside_queries_without_heads():
    torch.manual_seed(2)
    key = torch.randn(2, 5, 3, 16, device="cuda").bfloat16()
    query = torch.zeros(2, 5, 0, 16, device="cuda").bfloat16()
    q, k = nb.rotary(query, key)
    assert q.shape == query.shape and torch.equal(k, nb.rotary(key))
    leaf, none = key.clone().requires_grad_(), query.clone().requires_grad_()
    d = torch.randn_like(key)
    want, = torch.autograd.grad(nb.rotary(leaf), leaf, d)
    a, b = nb.rotary(none, leaf)
    got = torch.autograd.grad((a, b), (none, leaf), (torch.zeros_like(a), d))
    assert got[0].shape == query.shape and torch.equal(got[1], want)


def _assert_holds(got, x):
    """8-bit rows read back against what was written: half an e4m3 step of each value (at the row's scale the
    smallest step is 2**-9), and two half steps of bf16 for products that torch splits differently."""
    x = x.float()
    scale = x.abs().amax(-1, keepdim=True) / 448
    tol = torch.maximum(x.abs() * 2.0 ** -4, 2.0 ** -10 * scale) * 1.01 + 2 * 2.0 ** -8 * x.abs().amax(-1, keepdim=True)
    assert ((got - x).abs() <= tol).all()


@pytest.mark.parametrize("rotary_theta", [None, 1e4])
@pytest.mark.parametrize("kernel_size,dilation", [(24, 1), (7, 4), (100, 1)])
def test_steps_of_a_layer_over_an_eight_bit_cache(kernel_size, dilation, rotary_theta):
    """The layer's steps against 64 bits on the cache as it was quantised: no tolerance for the 8 bits."""
    torch.manual_seed(3)
    B, N, heads, dim = 3, 120, 4, 32
    layer = nb.NeighborhoodAttention1D(heads * dim, heads, kernel_size, 1, dilation, True,
                                       rotary_theta=rotary_theta).cuda().bfloat16().eval()
    x = torch.randn(B, N, heads * dim, device="cuda").bfloat16()
    cache = nb.KVCache.allocate(60, 8, heads, dim, E4M3)
    table = torch.randperm(60, device="cuda")[:B * 15].view(B, 15).int()
    at = [60, 31, 45]
    weight, bias = layer.proj.weight.detach().double().cpu(), layer.proj.bias.detach().double().cpu()
    half = ref.HALF_STEP[torch.bfloat16]
    with torch.no_grad():
        q_all, k_all, v_all = layer._project(x)              # at the positions of the layout
        layer.prefill(x[:, :60].contiguous(), cache, table, torch.tensor(at, dtype=torch.int32, device="cuda"))
        for tokens in (1, 3, 1, 2):
            rows = torch.stack([x[b, at[b]:at[b] + tokens] for b in range(B)])
            q = torch.stack([q_all[b, at[b]:at[b] + tokens] for b in range(B)])
            at = [n + tokens for n in at]
            lengths = torch.tensor(at, dtype=torch.int32, device="cuda")
            y = layer.decode(rows, cache, table, lengths).double().cpu()
            key, value = nb.kv_cache_read(cache, table, max(at), dtype=torch.float32)
            for b in range(B):
                _assert_holds(key[b, :at[b]], k_all[b, :at[b]])
                _assert_holds(value[b, :at[b]], v_all[b, :at[b]])
            # the projection of a few rows may be summed in another order than that of all: its own queries
            positions = (lengths[:, None] - tokens + torch.arange(tokens, device="cuda", dtype=torch.int32))[..., None]
            own = layer._project(rows, positions if rotary_theta else None)[0]
            assert (own.float() - q.float()).abs().max() <= 4 * half * q.float().abs().max()
            cpu = nb.KVCache(*(t.cpu() for t in cache))
            out, _, tol, _ = ref.decode(own.cpu(), cpu, table.cpu(), at, kernel_size, dilation, layer.scale, 2.0 ** -11)
            out, tol = out.flatten(2), tol.flatten(2)
            want = out @ weight.T + bias
            # the attention's own error through the weights, the result's half step, and two more of the sum
            # of magnitudes where torch adds partial sums in the type
            over = tol @ weight.abs().T + half * want.abs() + 2 * half * (out.abs() @ weight.abs().T)
            assert ((y - want).abs() <= over).all()
            # (an attention of zeros would be told apart, for every token)
            assert ((want - bias).abs() > 2 * over).any(-1).all()


def test_a_run_over_an_eight_bit_cache():
    """Rotary positions, writes and attention of one model step after the other, against 64 bits on the cache
    as it was quantised."""
    torch.manual_seed(9)
    B, N, heads, heads_kv, dim, at = 2, 90, 4, 2, 64, 70
    q, k, v = (torch.randn(B, N, h, dim, device="cuda").bfloat16() for h in (heads, heads_kv, heads_kv))
    qr, kr = nb.rotary(q, k)
    cache = nb.KVCache.allocate(30, 8, heads_kv, dim, E4M3)
    table = torch.randperm(30, device="cuda")[:24].view(B, 12).int()
    nb.kv_cache_write(cache, kr[:, :at], v[:, :at], table)
    for tokens in (1, 1, 4, 1, 8, 1, 4):
        start = torch.full((B,), at, dtype=torch.int32, device="cuda")
        positions = (start[:, None] + torch.arange(tokens, device="cuda", dtype=torch.int32))[..., None]
        qs, ks = nb.rotary(q[:, at:at + tokens], k[:, at:at + tokens], positions=positions)
        nb.kv_cache_write(cache, ks, v[:, at:at + tokens], table, start)
        at += tokens
        assert torch.equal(qs, qr[:, at - tokens:at])
        out, _ = _check(qs, cache, table, start + tokens, 32)
        key, value = nb.kv_cache_read(cache, table, at, dtype=torch.float32)
        _assert_holds(key, kr[:, :at])
        _assert_holds(value, v[:, :at])
        assert (out.float().abs() > 0.1).any(-1).all()
    assert at == N


@pytest.mark.parametrize("heads", [4, 24])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("octaves", [12, 18])
def test_query_channels_of_very_different_size(dtype, heads, octaves):
    """8-bit keys that are zero in the query's largest channels, so that the small ones decide. Within 2**13 of
    a row's largest channel nothing is lost of a bf16 query; below, and of fp16 queries, 2**-21 of the largest."""
    q, cache, table, n = _state(dtype, E4M3, [90, 33], 2, heads, 2, 64, 16)
    size = 2.0 ** (2 - octaves * torch.arange(64, device="cuda") / 63)
    q = ((1 + torch.rand(q.shape, device="cuda")) * torch.sign(q.float()) * size).to(dtype)
    key = torch.randn(2, 90, 2, 64, device="cuda").to(dtype)
    key[..., :20] = 0
    value = torch.randn(2, 90, 2, 64, device="cuda").to(dtype)
    nb.kv_cache_write(cache, key, value, table, counts=n)
    scale = 2.0 ** 4
    out, lse = nb.na1d_decode(q, cache, table, n, scale=scale, return_lse=True)
    cpu = nb.KVCache(*(t.cpu() for t in cache))
    want, want_lse, tol, tol_lse = ref.decode(q.cpu(), cpu, table.cpu(), n.tolist(), 0, 1, scale, 2.0 ** -11)
    lost = 0.0 if octaves <= 12 and dtype == torch.bfloat16 else 2.0 ** -21
    key = nb.kv_cache_read(cache, table, 90, counts=n, dtype=torch.float32)[0]
    logit = (lost * scale * q.float().abs().amax() * key.abs().sum(-1).max()).item()
    ref.assert_close(out, want, tol + 4 * logit * 8.0)      # (values below 8)
    ref.assert_close(lse, want_lse, tol_lse + logit)


@pytest.mark.parametrize("eight_bits", [False, True])
def test_counts_far_below_zero(eight_bits):
    """Nothing is written, and nothing read of the keys behind the call's tokens (whose number is no multiple of
    a block's)."""
    cache = nb.KVCache.allocate(40, 64, 2, 16, E4M3 if eight_bits else torch.bfloat16)
    for t in cache:
        if t is not None:
            t.copy_(torch.ones(t.shape, device="cuda").to(t.dtype))
    table = torch.arange(40, dtype=torch.int32, device="cuda").view(1, 40)
    x = torch.randn(1, 2501, 2, 16, device="cuda").bfloat16()
    for count in (-2 ** 31, -2 ** 31 + 1, -1):
        n = torch.tensor([count], dtype=torch.int32, device="cuda")
        nb.kv_cache_write(cache, x, x, table, counts=n)
        assert all((t.float() == 1).all() for t in cache if t is not None)
        assert not any(t.any() for t in nb.kv_cache_read(cache, table, 2501, counts=n))


def test_the_longest_read():
    """2**31 - 1 tokens, the last number that is accepted: what is cached, then zeros to the end."""
    cache = nb.KVCache.allocate(2, 8, 1, 1, torch.float16)
    for t in cache[:2]:
        t.copy_(torch.arange(1, 17, device="cuda").view(2, 8, 1, 1))
    table = torch.tensor([[1, 0, -1]], dtype=torch.int32, device="cuda")
    start = torch.tensor([3], dtype=torch.int32, device="cuda")
    key, value = nb.kv_cache_read(cache, table, 2 ** 31 - 1, start)
    want = torch.cat((torch.arange(12, 17), torch.arange(1, 9))).half().cuda()
    for t in (key, value):
        assert t.shape == (1, 2 ** 31 - 1, 1, 1) and torch.equal(t[0, :13, 0, 0], want)
        assert not t[0, 13:].any()


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("dim", [64, 33])
def test_rows_that_attend_nothing_in_either_part_merge_to_zeros(dtype, dim):
    """Attention over two caches joined: a place that a sequence does not have is empty in both."""
    q, one, table, n = _state(dtype, dtype, [1, 40, 0], 3, 4, 2, dim, 16)
    _, two, other, m = _state(dtype, dtype, [2, 0, 0], 3, 4, 2, dim, 16, seed=1)
    a, la = nb.na1d_decode(q, one, table, n, return_lse=True)
    b, lb = nb.na1d_decode(q, two, other, m, return_lse=True)
    for x, y, lx, ly in ((a, b, la, lb), (b, a, lb, la)):
        out, lse = nb.merge_attentions([x, y], [lx, ly])
        empty = torch.isneginf(la) & torch.isneginf(lb)
        assert empty[0, 0].all() and empty[2].all() and int(empty.sum()) == 4 * 4
        assert not out[empty].any() and torch.isneginf(lse[empty]).all()
        assert torch.isfinite(out).all() and torch.isfinite(lse[~empty]).all()
        assert torch.equal(out[1], a[1]) and torch.equal(lse[1], la[1])        # (nothing in the other part)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("dim,kernel_size,dilation,tokens", [(64, 24, 1, 200), (64, 7, 4, 200), (128, 100, 1, 90),
                                                             (33, 64, 1, 200)])
def test_what_lies_behind_a_prompt_does_not_reach_it(dtype, dim, kernel_size, dilation, tokens):
    """Padding that is not finite (memory that nothing was written to) changes no bit of the prompts' rows and of the
    cache."""
    torch.manual_seed(4)
    layer = nb.NeighborhoodAttention1D(2 * dim, 2, kernel_size, 1, dilation, True,
                                       rotary_theta=None if dim % 2 else 1e4).cuda().to(dtype).eval()
    counts = [tokens // 2, 17, tokens, 0]
    x = torch.randn(4, tokens, 2 * dim, device="cuda").to(dtype)
    n = torch.tensor(counts, dtype=torch.int32, device="cuda")
    table = torch.arange(56, device="cuda").int().view(4, 14)
    got = []
    for pad in (None, math.nan, math.inf):
        z = x.clone()
        for b in range(4):
            if pad is not None:
                z[b, counts[b]:] = pad
        given = z.clone()
        cache = nb.KVCache.allocate(56, 16, 2, dim, dtype)
        with torch.no_grad():
            y = layer.prefill(z, cache, table, n)
        assert torch.equal(z.nan_to_num(7.0), given.nan_to_num(7.0))
        rows = torch.cat([y[b, :counts[b]] for b in range(4)])
        got.append((rows, *nb.kv_cache_read(cache, table, tokens, counts=n)))
    for other in got[1:]:
        assert all(torch.equal(a, b) for a, b in zip(got[0], other))
    assert torch.isfinite(got[0][0]).all()
