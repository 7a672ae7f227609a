"""Plain 64-bit forms of the operators around a key/value cache, and the error that rounding allows them."""
import math

import torch

HALF_STEP = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8,
             torch.float8_e4m3fn: 2.0 ** -4}
E4M3_MAX, SMALLEST_SCALE = 448.0, 2.0 ** -126


# ---- rotary positions ------------------------------------------------------------------------------

def rotary(x, dims, theta, scale, positions, interleaved, inverse=False):
    """x [B, *X, H, D]; positions [B or 1, *X, axes] (float64)."""
    x = x.double()
    y, at = x.clone(), 0
    for a, dim in enumerate(dims):
        for i in range(dim // 2):
            one, two = (at + 2 * i, at + 2 * i + 1) if interleaved else (at + i, at + dim // 2 + i)
            angle = positions[..., a] * (scale[a] * theta[a] ** (-2.0 * i / dim))
            c, s = torch.cos(angle)[..., None], torch.sin(angle)[..., None]
            s = -s if inverse else s
            u, w = x[..., one], x[..., two]
            y[..., one], y[..., two] = u * c - w * s, u * s + w * c
        at += dim
    return y


def grid_positions(sides, origin):
    axes = [torch.arange(n, dtype=torch.float64) + o for n, o in zip(sides, origin)]
    return torch.stack(torch.meshgrid(*axes, indexing="ij"), -1)[None]


def rotary_tolerance(x, want, dims, interleaved, dtype):
    """A half step of the result, and the 32-bit sine and cosine (2 units in the last place of 1 each:
    2**-22 with the reduced angle's own rounding), products and their sum: 2**-21 of the pair's length."""
    pair, at = x.double().abs(), 0
    length = torch.zeros_like(pair)
    for dim in dims:
        for i in range(dim // 2):
            one, two = (at + 2 * i, at + 2 * i + 1) if interleaved else (at + i, at + dim // 2 + i)
            length[..., one] = length[..., two] = torch.hypot(pair[..., one], pair[..., two])
        at += dim
    return HALF_STEP[dtype] * want.abs() + 2.0 ** -21 * length + 2.0 ** -25


# ---- the cache ---------------------------------------------------------------------------------------

def quantise(x):
    """(values before they are rounded to e4m3, scale), 64 bits."""
    scale = (x.double().abs().amax(-1) / E4M3_MAX).clamp_min(SMALLEST_SCALE)
    return x.double() / scale[..., None], scale


def cached_rows(pages, scales, table_row, positions):
    """Rows [n, H, D] (float64) of the tokens at `positions`, and which of them are on a page."""
    ps, there = pages.shape[1], []
    rows = torch.zeros(len(positions), *pages.shape[2:], dtype=torch.float64)
    for i, p in enumerate(positions):
        page = int(table_row[p // ps]) if p >= 0 and p // ps < len(table_row) else -1
        ok = 0 <= page < pages.shape[0]
        there.append(ok)
        if ok:
            rows[i] = pages[page, p % ps].double()
            if scales is not None:
                rows[i] *= scales[page, p % ps].double()[:, None]
    return rows, torch.tensor(there, dtype=torch.bool)


# ---- decode --------------------------------------------------------------------------------------------

def decode(query, cache, table, lengths, kernel_size, dilation, scale, weight_step):
    """(out, lse, tolerance of out, tolerance of lse), all on the CPU in 64 bits. weight_step: half a
    step of the type that the weights are rounded to before the products with the values.

    Errors that add up: half a step of the result; the weights' rounding; the logits', whose 32-bit sums
    of D products and factors are off by (D + 8) 2**-24 of the sum of magnitudes; 32-bit sums over the n
    tokens; the exponentials' 2**-21. A weight that falls below the 16-bit type's normal numbers is off by
    up to 2**-25 of the largest one."""
    B, T, Hq, D = query.shape
    key, value, key_scale, value_scale = cache
    group = Hq // key.shape[2]
    out = torch.zeros(B, T, Hq, D, dtype=torch.float64)
    lse = torch.full((B, T, Hq), -math.inf, dtype=torch.float64)
    tol, tol_lse = torch.zeros_like(out), torch.zeros_like(lse)
    for b in range(B):
        n = int(lengths[b])
        for t in range(T):
            p = n - T + t
            if p < 0:
                continue
            at = list(range(p, -1, -dilation))
            at = at[:kernel_size] if kernel_size else at
            k, ok = cached_rows(key, key_scale, table[b], at)
            v, _ = cached_rows(value, value_scale, table[b], at)
            if not ok.any():
                continue
            k, v = (x[ok].repeat_interleave(group, 1) for x in (k, v))
            q = query[b, t].double()
            logits = scale * (q[None] * k).sum(-1)                  # [n, Hq]
            size = scale * (q[None] * k).abs().sum(-1)
            w = torch.softmax(logits, 0)
            lse[b, t] = torch.logsumexp(logits, 0)
            out[b, t] = (w[..., None] * v).sum(0)
            spread = (w[..., None] * v.abs()).sum(0)
            largest = (w[..., None] * v.abs()).amax((0, 2))[:, None]
            logit = (D + 8) * 2.0 ** -24 * (size.amax(0) + logits.abs().amax(0))
            tol_lse[b, t] = logit + (len(at) * 2.0 ** -24 + 2.0 ** -20) + 2.0 ** -23 * lse[b, t].abs()
            rel = 2 * weight_step + 4 * logit + len(at) * 2.0 ** -23 + 2.0 ** -19
            tol[b, t] = (HALF_STEP[query.dtype] * out[b, t].abs() + rel[:, None] * spread
                         + len(at) * 2.0 ** -24 * largest + 2.0 ** -25)
    return out, lse, tol, tol_lse


def assert_close(got, want, tol):
    got = got.double().cpu()
    finite = torch.isfinite(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    rest = ~finite & ~torch.isnan(want)
    assert torch.equal(got[rest], want[rest])
    over = ((got - want).abs() - tol)[finite]
    assert over.numel() == 0 or over.max() <= 0, (over.max().item(), int((over > 0).sum()))
