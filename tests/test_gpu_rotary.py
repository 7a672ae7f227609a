"""Rotary positions on the GPU against a plain 64-bit form: layouts, types, strides, positions, gradients."""
import pytest
import torch

import natten_b200 as nb
import natten_b200._lib as L
import serving_reference as ref
from natten_b200 import ops

pytestmark = pytest.mark.gpu


def _check(x, got, dims, theta, scale, positions, interleaved, inverse=False):
    x = x.detach().cpu()
    want = ref.rotary(x, dims, theta, scale, positions, interleaved, inverse)
    assert got.shape == x.shape and got.dtype == x.dtype and got.is_contiguous()
    ref.assert_close(got, want, ref.rotary_tolerance(x, want, dims, interleaved, x.dtype))


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("batch,sides,heads,heads_kv,dim,dims", [
    (1, (1,), 1, 0, 2, None),
    (3, (37,), 4, 2, 64, None),
    (2, (5, 9), 3, 3, 80, None),
    (1, (3, 5, 7), 6, 2, 128, None),
    (1, (3, 4, 5), 2, 1, 128, (44, 42, 42)),       # halves of 22 and 21 channels
    (2, (6, 5), 2, 2, 48, (8, 0)),                  # an axis without channels, channels without an axis
    (2, (11,), 2, 1, 33, (6,)),                     # an odd head
    (1, (700,), 2, 2, 256, None),
    (1, (4099,), 1, 1, 32, (16,)),                  # several tokens a block, a ragged last block
])
def test_layouts_and_types(dtype, interleaved, batch, sides, heads, heads_kv, dim, dims):
    torch.manual_seed(1)
    q = torch.randn(batch, *sides, heads, dim).to(dtype).cuda()
    k = torch.randn(batch, *sides, heads_kv, dim).to(dtype).cuda() if heads_kv else None
    theta = [10000.0, 500.0, 1e6][:len(sides)]
    scale = [1.0, 0.5, 3.0][:len(sides)]
    origin = [5, -3, 1000][:len(sides)]
    got = nb.rotary(q, k, dims, theta, origin=origin, position_scale=scale, interleaved=interleaved)
    dims = dims or nb.rotary_axis_dims(dim, len(sides))
    at = ref.grid_positions(sides, origin)
    for x, y in ((q, got if k is None else got[0]), (k, None if k is None else got[1])):
        if x is not None:
            _check(x, y, dims, theta, scale, at, interleaved)


@pytest.mark.parametrize("kind", [torch.int32, torch.int64, torch.float32])
@pytest.mark.parametrize("batched", [False, True])
@pytest.mark.parametrize("axes", [1, 3])
def test_given_positions_far_out(kind, batched, axes):
    torch.manual_seed(2)
    q = torch.randn(3, 50, 4, 64).cuda()
    k = torch.randn(3, 50, 1, 64).cuda()
    at = torch.randint(-2 ** 20, 2 ** 20, (3 if batched else 1, 50, axes)).to(kind)
    if kind == torch.float32:
        at = at + 0.25
    if kind == torch.int64:
        at = at * 2 ** 12
    got = nb.rotary(q, k, positions=at.cuda())
    dims = nb.rotary_axis_dims(64, axes)
    # what 64 bits lose of an angle of up to 2**32: 2**-52 of it on either side, with the frequency's
    # rounding 2**-18 at most, against 2**-9 (2**12 times that) of a 32-bit angle
    far = 2.0 ** -17 if kind == torch.int64 else 0.0
    for x, y in ((q, got[0]), (k, got[1])):
        want = ref.rotary(x.cpu(), dims, [1e4] * axes, [1.0] * axes, at.double(), False)
        tol = ref.rotary_tolerance(x.cpu(), want, dims, False, x.dtype) + far * 8
        ref.assert_close(y, want, tol)


@pytest.mark.parametrize("interleaved", [False, True])
def test_views_in_any_strides(interleaved):
    torch.manual_seed(3)
    dims = nb.rotary_axis_dims(64, 2)
    at = ref.grid_positions((6, 7), (0, 0))
    fused = torch.randn(2, 6, 7, 3, 4, 64).bfloat16().cuda()
    flat = torch.randn(2 * 6 * 7 * 4 * 66 + 3).bfloat16().cuda()
    views = [
        fused.unbind(-3)[0],                                                        # of a fused projection
        torch.randn(2, 4, 6, 7, 64).bfloat16().cuda().permute(0, 2, 3, 1, 4),       # heads first
        torch.randn(2, 6, 7, 4, 64, 2).bfloat16().cuda()[..., 0],                   # channels apart
        torch.randn(2, 6, 7, 64, 4).bfloat16().cuda().transpose(-1, -2),
        torch.randn(1, 1, 7, 4, 64).bfloat16().cuda().expand(2, 6, 7, 4, 64),       # broadcast
        flat[3:].as_strided((2, 6, 7, 4, 64), (6 * 7 * 4 * 66, 7 * 4 * 66, 4 * 66, 66, 1)),
        flat[1:].as_strided((2, 6, 7, 4, 64), (6 * 7 * 4 * 64, 7 * 4 * 64, 4 * 64, 64, 1)),
    ]
    for v in views:
        for w in views:
            a, b = nb.rotary(v, w, interleaved=interleaved)
            for x, y in ((v, a), (w, b)):
                _check(x, y, dims, [1e4] * 2, [1.0] * 2, at, interleaved)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("interleaved", [False, True])
def test_gradients_are_the_turn_back(dtype, interleaved):
    torch.manual_seed(4)
    sides, dims = (5, 6), [24, 32]
    q = torch.randn(2, *sides, 3, 64).to(dtype).cuda().requires_grad_()
    k = torch.randn(1, 1, sides[1], 1, 64).to(dtype).cuda().requires_grad_()     # broadcast before the call
    a, b = nb.rotary(q, k.expand(2, *sides, 1, 64), dims, interleaved=interleaved)
    da, db = torch.randn_like(a), torch.randn_like(b)
    gq, gk = torch.autograd.grad((a, b), (q, k), (da, db))
    at = ref.grid_positions(sides, (0, 0))
    _check(da, gq, dims, [1e4] * 2, [1.0] * 2, at, interleaved, inverse=True)
    rows = ref.rotary(db.cpu(), dims, [1e4] * 2, [1.0] * 2, at, interleaved, inverse=True)
    want = rows.sum((0, 1), keepdim=True)
    # ten rows, each rounded to the type, summed in the type by autograd of expand
    tol = ref.HALF_STEP[dtype] * 12 * rows.abs().sum((0, 1), keepdim=True) + 2.0 ** -18
    ref.assert_close(gk, want, tol)
    # one of the two alone; an output that nothing uses; strided gradients
    only, = torch.autograd.grad(nb.rotary(q, k.detach().expand(2, *sides, 1, 64), dims,
                                          interleaved=interleaved)[0], q, da)
    assert torch.equal(only, gq)
    out_k = nb.rotary(q.detach(), q, dims, interleaved=interleaved)[1]
    g, = torch.autograd.grad(out_k, q, da.transpose(1, 2).contiguous().transpose(1, 2))
    assert torch.equal(g, gq)
    g, = torch.autograd.grad(nb.rotary(q, None, dims, interleaved=interleaved).sum(), q)
    _check(torch.ones_like(q), g, dims, [1e4] * 2, [1.0] * 2, at, interleaved, inverse=True)


def test_gradient_against_differences_and_second_derivative():
    torch.manual_seed(5)
    q = torch.randn(1, 4, 2, 8).cuda().requires_grad_()
    k = torch.randn(1, 4, 1, 8).cuda().requires_grad_()
    at = torch.randint(0, 50, (1, 4, 2), device="cuda")
    w = torch.randn(1, 4, 2, 8).cuda()

    def f(q, k):
        a, b = nb.rotary(q, k, positions=at)
        return (a * a * w).sum() + (b ** 3).sum()

    gq, gk = torch.autograd.grad(f(q, k), (q, k), create_graph=True)
    for x, g in ((q, gq), (k, gk)):
        for i in (0, 3, 9, 30):
            step = torch.zeros_like(x).flatten()
            step[i] = 2.0 ** -7
            step = step.view_as(x)
            args = [(q + step, k), (q - step, k)] if x is q else [(q, k + step), (q, k - step)]
            d = (f(*args[0]) - f(*args[1])).item() / 2.0 ** -6
            # the third derivative's term (6 2**-14 / 6 at most) and 32-bit sums of about 100
            assert abs(d - g.flatten()[i].item()) <= 2.0 ** -13 + 100 * 2.0 ** -22 * 2.0 ** 6
    # sum w a^2 is a quadratic form: its Hessian times v is the gradient at v
    v = torch.randn_like(q)
    hv, = torch.autograd.grad(gq, q, v, retain_graph=True)
    gv, = torch.autograd.grad(f(v.requires_grad_(), k.detach()), v)
    assert (hv - gv).abs().max() <= 1e-4
    assert torch.autograd.grad(gk, k, torch.ones_like(k))[0].abs().max() > 0


def test_non_finite_values_stay_in_their_pair():
    x = torch.ones(1, 9, 2, 16).cuda()
    x[0, 4, 1, 3] = float("nan")
    x[0, 6, 0, 15] = float("inf")
    y = nb.rotary(x, axis_dims=(16,))
    bad = ~torch.isfinite(y)
    at = {(4, 1, 3), (4, 1, 11), (6, 0, 7), (6, 0, 15)}
    assert {tuple(i[1:]) for i in bad.nonzero().tolist()} == at


def test_empty_other_stream_and_captured():
    q = torch.zeros(0, 4, 2, 16).cuda()
    assert nb.rotary(q).shape == q.shape
    assert nb.rotary(torch.zeros(2, 0, 2, 16).cuda(), torch.zeros(2, 0, 1, 16).cuda())[1].shape == (2, 0, 1, 16)
    torch.manual_seed(6)
    q = torch.randn(2, 33, 4, 64).bfloat16().cuda()
    at = torch.arange(66, device="cuda").view(2, 33, 1)
    want = nb.rotary(q, positions=at)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = nb.rotary(q, positions=at)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    x, p = q.clone(), at.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = nb.rotary(x, positions=p)
    for shift in (0, 7):
        x.copy_(q * (1 + shift))
        p.copy_(at + shift)
        graph.replay()
        assert torch.equal(out, nb.rotary(x, positions=p))


def test_captured_training_step():
    torch.manual_seed(7)
    q = torch.randn(1, 40, 2, 32).cuda().requires_grad_()
    d = torch.randn(1, 40, 2, 32).cuda()
    want, = torch.autograd.grad(nb.rotary(q), q, d)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.autograd.grad(nb.rotary(q), q, d)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        g, = torch.autograd.grad(nb.rotary(q), q, d)
    graph.replay()
    assert torch.equal(g, want)


def test_op_and_compile():
    torch.manual_seed(8)
    q = torch.randn(2, 5, 6, 4, 64).bfloat16().cuda()
    k = torch.randn(2, 5, 6, 2, 64).bfloat16().cuda()
    tests = ("test_schema", "test_faketensor", "test_autograd_registration")
    how = ([32, 32], [1e4, 1e4], [1.0, 1.0], [0, 0], None, False, False)
    torch.library.opcheck(ops.rotary, (q.clone().requires_grad_(), k, *how), test_utils=tests)
    torch.library.opcheck(ops.rotary, (q, None, *how), test_utils=tests)

    def f(q, k):
        a, b = nb.rotary(q * 1.0, k, interleaved=True)
        return a.float() + 1.0, b

    want = f(q, k)
    got = torch.compile(f, fullgraph=True)(q, k)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    leaf = q.clone().requires_grad_()
    (g,) = torch.autograd.grad(torch.compile(f, fullgraph=True)(leaf, k)[0].sum(), leaf)
    (h,) = torch.autograd.grad(f(leaf, k)[0].sum(), leaf)
    assert torch.equal(g, h)
    assert L.device_status() == 0


def test_native_front_and_registered_operators_give_the_same(monkeypatch):
    import natten_b200.positions as module
    torch.manual_seed(10)
    q = torch.randn(2, 5, 6, 4, 64).bfloat16().cuda().requires_grad_()
    k = torch.randn(2, 5, 6, 2, 64).bfloat16().cuda().requires_grad_()
    dq, dk = torch.randn_like(q), torch.randn_like(k)
    at = torch.randint(0, 99, (1, 5, 6, 3), device="cuda")
    for kw in ({}, {"positions": at}, {"axis_dims": [8, 24], "theta": (10, 1e5), "origin": (3, -1),
                                       "position_scale": (2, 0.5), "interleaved": True}):
        got = []
        for native in (True, False):
            monkeypatch.setattr(module, "_native_eligible", lambda native=native: native)
            a, b = nb.rotary(q, k, **kw)
            got.append((a, b, nb.rotary(q.detach(), **kw), *torch.autograd.grad((a, b), (q, k), (dq, dk)),
                        torch.autograd.grad(nb.rotary(q, k.detach(), **kw)[0], q, dq)[0],
                        torch.autograd.grad(nb.rotary(q.detach(), k, **kw)[1], k, dk)[0]))
        for x, y in zip(*got):
            assert torch.equal(x, y)
    # the gradients of both operands in one launch
    monkeypatch.setattr(module, "_native_eligible", lambda: True)
    a, b = nb.rotary(q, k)
    before = L.launches
    torch.autograd.grad((a, b), (q, k), (dq, dk))
    assert L.launches == before + 1


@pytest.mark.parametrize("given", [False, True])
@pytest.mark.parametrize("batch,sides,heads,heads_kv,dim", [
    (70, (6, 50), 2, 1, 64),          # batch entries that share a block, the last group of them ragged
    (33, (5, 9, 30), 3, 0, 48),
    (64, (641,), 1, 1, 16),
    (300, (1,), 2, 2, 32),
])
def test_batch_entries_share_their_angles(given, batch, sides, heads, heads_kv, dim):
    torch.manual_seed(11)
    q = torch.randn(batch, heads, *sides, dim).half().cuda().movedim(1, -2)
    k = torch.randn(batch, *sides, heads_kv, dim).half().cuda() if heads_kv else None
    at = ref.grid_positions(sides, [0] * len(sides))
    kw = {}
    if given:
        at = torch.randint(0, 1000, (1, *sides, 2)).double()
        kw = {"positions": at.int().cuda()}
    dims = [2 * (dim // 8), 2 * (dim // 16), 0][:at.shape[-1]]       # the rest passes through
    got = nb.rotary(q, k, dims, **kw)
    theta, scale = [1e4] * len(dims), [1.0] * len(dims)
    _check(q, got if k is None else got[0], dims, theta, scale, at, False)
    if k is not None:
        _check(k, got[1], dims, theta, scale, at, False)
    # positions of each batch entry's own, the same ones: the same bits
    if given:
        own = nb.rotary(q, k, dims, positions=kw["positions"].expand(batch, *sides, 2))
        for x, y in zip((got,) if k is None else got, (own,) if k is None else own):
            assert torch.equal(x, y)
