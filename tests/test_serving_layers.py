"""Layers with rotary positions, and the causal 1-D layer served from a paged cache."""
import pytest
import torch

import natten_b200 as nb
import serving_reference as ref


def test_layer_arguments():
    layer = nb.NeighborhoodAttention2D(64, 2, 5, rotary_theta=(1e4, 100.0), rotary_axis_dims=(8, 24))
    assert set(layer.state_dict()) == set(nb.NeighborhoodAttention2D(64, 2, 5).state_dict())
    assert "rotary_theta" in repr(layer) and "rotary" not in repr(nb.NeighborhoodAttention2D(64, 2, 5))
    for kw in ({"rotary_theta": 0.0}, {"rotary_theta": 1e4, "rotary_axis_dims": (8,)},
               {"rotary_theta": 1e4, "rotary_axis_dims": (32, 8)}, {"rotary_theta": "far"}):
        with pytest.raises(ValueError):
            nb.NeighborhoodAttention2D(64, 2, 5, **kw)


def test_modules_pickled_before_there_were_positions():
    layer = nb.NeighborhoodAttention2D(64, 2, 5)
    state = {n: v for n, v in layer.__dict__.items() if not n.startswith("rotary")}
    old = nb.NeighborhoodAttention2D.__new__(nb.NeighborhoodAttention2D)
    old.__dict__.update(state)
    assert repr(old) == repr(layer) and old.rotary_theta is None


def test_serving_refusals():
    x = torch.zeros(2, 3, 64)
    cache = nb.KVCache.allocate(4, 8, 2, 32, torch.float32, device="cpu")
    table, n = torch.zeros(2, 2, dtype=torch.int32), torch.tensor([3, 3], dtype=torch.int32)
    for layer in (nb.NeighborhoodAttention1D(64, 2, 5), nb.NeighborhoodAttention1D(64, 2, 5, 2, is_causal=True)):
        with pytest.raises(ValueError):
            layer.decode(x, cache, table, n)
        with pytest.raises(ValueError):
            layer.prefill(x, cache, table)
    layer = nb.NeighborhoodAttention1D(64, 2, 5, is_causal=True)
    with pytest.raises(ValueError):
        layer.decode(x[0], cache, table, n)
    with pytest.raises(NotImplementedError):                     # parameters with gradients
        layer.prefill(x, cache, table)
    with torch.no_grad(), pytest.raises(RuntimeError):           # CPU tensors
        layer.prefill(x, cache, table)


@pytest.mark.gpu
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("cls,shape,ks,dims", [
    (nb.NeighborhoodAttention1D, (150,), 33, None),
    (nb.NeighborhoodAttention2D, (14, 18), (5, 7), (8, 48)),
    (nb.NeighborhoodAttention3D, (6, 8, 10), (3, 4, 5), None),
])
def test_layers_with_rotary_positions(cls, shape, ks, dims, interleaved):
    """Projection, rotary positions, attention, projection: the layer is these, forward and backward."""
    torch.manual_seed(1)
    layer = cls(128, 2, ks, rotary_theta=500.0, rotary_axis_dims=dims, rotary_interleaved=interleaved)
    layer = layer.cuda().bfloat16()
    x = torch.randn(2, *shape, 128, device="cuda").bfloat16().requires_grad_()
    y = layer(x)
    q, k, v = layer.qkv(x).unflatten(-1, (3, 2, 64)).unbind(-3)
    q, k = nb.rotary(q, k, dims, 500.0, interleaved=interleaved)
    fn = {1: nb.na1d, 2: nb.na2d, 3: nb.na3d}[len(shape)]
    want = layer.proj(fn(q, k, v, ks).flatten(-2))
    assert torch.equal(y, want)
    d = torch.randn_like(y)
    params = [x, *layer.parameters()]
    for a, b in zip(torch.autograd.grad(y, params, d), torch.autograd.grad(want, params, d)):
        # the same kernels; sums over tokens in torch's matrix products may be split differently
        assert (a.float() - b.float()).abs().max() <= 4 * ref.HALF_STEP[torch.bfloat16] * b.float().abs().max()
    plain = cls(128, 2, ks).cuda().bfloat16()
    plain.load_state_dict(layer.state_dict())
    assert not torch.equal(plain(x), y)
    torch.compiler.reset()      # (other tests have compiled the layers' forward often)
    with torch.no_grad():
        compiled = torch.compile(layer, fullgraph=True)(x)
        assert torch.equal(compiled, layer(x))


@pytest.mark.gpu
@pytest.mark.parametrize("rotary_theta", [None, 1e4])
@pytest.mark.parametrize("dtype,cache_dtype", [(torch.bfloat16, torch.bfloat16), (torch.float16, torch.float16),
                                               (torch.float32, torch.float32),
                                               (torch.bfloat16, torch.float8_e4m3fn)])
@pytest.mark.parametrize("kernel_size,dilation", [(24, 1), (7, 4), (100, 1)])
def test_prompt_and_steps_give_what_the_whole_sequence_gives(dtype, cache_dtype, kernel_size, dilation,
                                                             rotary_theta):
    torch.manual_seed(2)
    B, N, heads, dim = 3, 120, 4, 32
    layer = nb.NeighborhoodAttention1D(heads * dim, heads, kernel_size, 1, dilation, True,
                                       rotary_theta=rotary_theta).cuda().to(dtype).eval()
    x = torch.randn(B, N, heads * dim, device="cuda").to(dtype)
    prompts = [60, 31, 45]
    cache = nb.KVCache.allocate(60, 8, heads, dim, cache_dtype)
    table = torch.randperm(60, device="cuda")[:B * 15].view(B, 15).int()
    counts = torch.tensor(prompts, dtype=torch.int32, device="cuda")
    # Values and outputs of the attention are averages of projections of unit size (uniform weights of
    # 1 / sqrt(E): about 0.6), below 4; the output projection sums E of them with weights below E^-0.5.
    # Each path rounds weights and outputs to the type twice; an 8-bit cache rounds values and logits by
    # half an e4m3 step.
    step = ref.HALF_STEP[dtype] if dtype != torch.float32 else 2.0 ** -18
    tol = 4 * 4 * step + (4 * 2.0 ** -4 if cache_dtype == torch.float8_e4m3fn else 0.0)
    with torch.no_grad():
        want = layer(x)
        y = layer.prefill(x[:, :60].contiguous(), cache, table, counts)
        for b in range(B):
            assert (y[b, :prompts[b]].float() - want[b, :prompts[b]].float()).abs().max() <= 4 * 4 * step
        at = counts.clone()
        for tokens in (1, 3, 1, 2):
            rows = torch.stack([x[b, int(at[b]):int(at[b]) + tokens] for b in range(B)])
            at += tokens
            y = layer.decode(rows, cache, table, at)
            for b in range(B):
                end = int(at[b])
                assert (y[b].float() - want[b, end - tokens:end].float()).abs().max() <= tol


@pytest.mark.gpu
def test_a_refused_prompt_leaves_the_cache_alone():
    layer = nb.NeighborhoodAttention1D(64, 2, 7, 1, 4, True).cuda().half().eval()
    cache = nb.KVCache.allocate(4, 8, 2, 32, torch.float16)
    for t in cache[:2]:
        t.zero_()
    table = torch.arange(4, device="cuda").int().view(1, 4)
    with torch.no_grad():
        with pytest.raises(ValueError):
            layer.prefill(torch.randn(1, 20, 64, device="cuda").half(), cache, table)      # 7 x 4 tokens
        with pytest.raises(ValueError):
            layer.decode(torch.randn(1, 1, 64, device="cuda").half(), cache, table,
                         torch.ones(1, dtype=torch.int64, device="cuda"))
    assert not cache.key.any() and not cache.value.any()


@pytest.mark.gpu
def test_captured_step_of_a_layer():
    """One decoding step as a CUDA graph, replayed for a whole continuation."""
    torch.manual_seed(3)
    B, heads, dim, prompt, steps = 2, 4, 64, 20, 12
    layer = nb.NeighborhoodAttention1D(heads * dim, heads, 16, is_causal=True, rotary_theta=1e4)
    layer = layer.cuda().bfloat16().eval()
    x = torch.randn(B, prompt + steps, heads * dim, device="cuda").bfloat16()
    caches = [nb.KVCache.allocate(20, 4, heads, dim) for _ in range(2)]
    table = torch.randperm(20, device="cuda")[:16].view(B, 8).int()
    with torch.no_grad():
        for c in caches:
            layer.prefill(x[:, :prompt].contiguous(), c, table)
        token, n = x[:, prompt:prompt + 1].clone(), torch.full((B,), prompt + 1, dtype=torch.int32, device="cuda")
        layer.decode(token, caches[0], table, n)                 # warm-up: the step that is replayed first
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = layer.decode(token, caches[0], table, n)
        for i in range(steps):
            token.copy_(x[:, prompt + i:prompt + i + 1])
            n.fill_(prompt + i + 1)
            graph.replay()
            want = layer.decode(token, caches[1], table, n)
            assert torch.equal(y, want)
        used = [nb.kv_cache_read(c, table, prompt + steps) for c in caches]
        assert torch.equal(used[0][0], used[1][0]) and torch.equal(used[0][1], used[1][1])
