"""The operators around attention that a served or trained model needs beside it, as a user's program
calls them: rotary positions over several token axes, the paged key/value cache (writing, reading
back) and attention of the newest tokens over that cache.

A case is a dict of plain values. Token layouts are texts such as "32x48x80".

  op       "decode" (na1d_decode), "write" (kv_cache_write), "read" (kv_cache_read), "rotary"
  dtype    of query, key and value; ``cache`` is the type the cache holds ("fp8": e4m3 with one fp32
           scale for each token and head)
  low, high  decode, read: the sequences' lengths run evenly from low to high (their order is random)
  new      decode: newest tokens of each sequence that are queries; write: tokens given to the call
  kernel   decode: tokens in the window, 0 for the whole sequence
  page     tokens of a page
"""
import math
import random

import torch

own = False

DTYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16,
          "fp8": torch.float8_e4m3fn}
BYTES = {"fp32": 4, "fp16": 2, "bf16": 2, "fp8": 1}
E4M3_MAX = 448.0
SMALLEST_SCALE = 2.0 ** -126


def _decode(name, dtype, cache, batch, new, heads, heads_kv, head_dim, low, high, kernel, page,
            dilation=1):
    return {"name": name, "op": "decode", "dtype": dtype, "cache": cache, "batch": batch, "new": new,
            "heads": heads, "heads_kv": heads_kv, "head_dim": head_dim, "low": low, "high": high,
            "kernel": kernel, "page": page, "dilation": dilation}


def _move(name, op, dtype, cache, batch, new, heads_kv, head_dim, low, high, page):
    return {"name": name, "op": op, "dtype": dtype, "cache": cache, "batch": batch, "new": new,
            "heads_kv": heads_kv, "head_dim": head_dim, "low": low, "high": high, "page": page}


def _rotary(name, dtype, batch, heads, heads_kv, tokens, head_dim, train=False, interleaved=False,
            explicit=False):
    return {"name": name, "op": "rotary", "dtype": dtype, "batch": batch, "heads": heads,
            "heads_kv": heads_kv, "tokens": tokens, "head_dim": head_dim, "train": train,
            "interleaved": interleaved, "explicit": explicit}


def listed():
    return [
        # One user's next token, grouped query heads, a sliding window: what the user waits for.
        _decode("decode-one", "bf16", "bf16", 1, 1, 16, 4, 128, 8190, 8190, 512, 64),
        # A step of a server: many sequences of very different lengths behind a sliding window.
        _decode("decode-window", "bf16", "bf16", 64, 1, 16, 4, 128, 1, 32768, 2048, 64),
        # A step with long contexts attended whole, the cache in 8 bits: the largest read.
        _decode("decode-long-fp8", "bf16", "fp8", 16, 1, 16, 4, 128, 4099, 32768, 0, 64),
        # Drafted tokens checked together, as many key heads as query heads, small pages.
        _decode("decode-drafts", "fp16", "fp16", 24, 5, 12, 12, 64, 700, 8190, 1000, 16),
        # Single precision, a dilated window, pages of odd size, a narrow head.
        _decode("decode-fp32-dilated", "fp32", "fp32", 8, 1, 6, 2, 48, 17, 4096, 300, 20, dilation=4),
        # The step's new token of each sequence goes into the cache.
        _move("write-step", "write", "fp16", "fp16", 64, 1, 4, 128, 1, 32768, 64),
        # Prompts of different lengths go into an 8-bit cache.
        _move("write-prompts-fp8", "write", "bf16", "fp8", 4, 8190, 4, 128, 2000, 8190, 64),
        # A short prefix read back in single precision.
        _move("read-short", "read", "fp32", "fp32", 2, 0, 2, 48, 300, 512, 20),
        # Prefixes read back out of an 8-bit cache, for dense attention of a long chunk over them.
        _move("read-prefixes-fp8", "read", "bf16", "fp8", 4, 0, 4, 128, 8190, 32768, 64),
        # Rotary positions of one new token of each sequence, positions given.
        _rotary("rotary-step", "bf16", 64, 16, 4, "1", 128, explicit=True),
        # Queries and keys of a video, views of the fused projection.
        _rotary("rotary-video", "bf16", 1, 24, 24, "32x48x80", 128),
        # A smaller video model in training, adjacent channels paired.
        _rotary("rotary-video-train", "bf16", 1, 12, 12, "15x30x52", 64, train=True, interleaved=True),
    ]


# ---- cases of the same ranges ---------------------------------------------------------------------

def _log(rng, lo, hi):
    """An integer between lo and hi, spread evenly over its logarithm."""
    return int(min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5)))))))


def draw(rng: random.Random):
    op = rng.choice(["decode", "decode", "decode", "write", "read", "rotary", "rotary"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    if op == "rotary":
        nd = rng.choice([1, 2, 3])
        sides = {1: lambda: [_log(rng, 1, 32768)],
                 2: lambda: [_log(rng, 7, 256) for _ in range(2)],
                 3: lambda: [_log(rng, 3, 32), _log(rng, 9, 60), _log(rng, 9, 80)]}[nd]()
        dim = rng.choice([32, 64, 80, 128])
        heads_kv = _log(rng, 1, 12)
        heads = heads_kv * rng.choice([1, 1, 2, 4])
        most = 32 * 48 * 80 * 48 * 128 // 2
        train = rng.random() < 0.5
        room = most // (math.prod(sides) * (heads + heads_kv) * dim * (2 if train else 1)
                        * (2 if dtype == "fp32" else 1))
        while room < 1:
            sides[0] = max(1, sides[0] // 2)
            room = most // (math.prod(sides) * (heads + heads_kv) * dim * (2 if train else 1)
                            * (2 if dtype == "fp32" else 1))
        return {"op": op, "dtype": dtype, "batch": _log(rng, 1, min(64, room)), "heads": heads,
                "heads_kv": heads_kv, "tokens": "x".join(str(s) for s in sides), "head_dim": dim,
                "train": train, "interleaved": rng.random() < 0.5, "explicit": rng.random() < 0.3}
    cache = "fp8" if rng.random() < 0.4 else dtype
    dim = rng.choice([48, 64, 80, 128, 128, 128])
    heads_kv = _log(rng, 1, 16)
    page = rng.choice([16, 20, 32, 64, 64, 128, 256])
    high = _log(rng, 16, 32768)
    most = 16 * 18433 * 4 * 128 // (4 if dtype == "fp32" else 1)    # elements of keys that are attended
    if op == "decode":
        new = rng.choice([1, 1, 1, 2, 4, 8])
        kernel = rng.choice([0, _log(rng, 16, 4096)])
        dilation = rng.choice([1, 1, 1, 2, 5]) if kernel else 1
        span = min(kernel or high, high)
        batch = _log(rng, 1, max(1, min(128, most // (span * heads_kv * dim * new))))
        return {"op": op, "dtype": dtype, "cache": cache, "batch": batch, "new": new,
                "heads": heads_kv * rng.choice([1, 2, 4, 7, 8]), "heads_kv": heads_kv,
                "head_dim": dim, "low": min(high, _log(rng, 1, high)), "high": high,
                "kernel": kernel, "page": page, "dilation": dilation}
    most //= 2
    batch = _log(rng, 1, max(1, min(64, most // (high * heads_kv * dim))))
    new = 0
    if op == "write":
        new = rng.choice([1, _log(rng, 1, high)])
    return {"op": op, "dtype": dtype, "cache": cache, "batch": batch, "new": new, "heads_kv": heads_kv,
            "head_dim": dim, "low": max(1, min(high, high // rng.choice([1, 2, 16]))), "high": high,
            "page": page}


# ---- inputs ------------------------------------------------------------------------------------------

def _lengths(case):
    n, lo, hi = case["batch"], case["low"], case["high"]
    return [hi if n == 1 else lo + (hi - lo) * i // (n - 1) for i in range(n)]


def _sides(case):
    return [int(x) for x in case["tokens"].split("x")]


def _quantise(x):
    """e4m3 values and one scale for each row of the last axis: the largest magnitude becomes 448."""
    scale = (x.abs().amax(-1) / E4M3_MAX).clamp_min(SMALLEST_SCALE)
    return (x / scale[..., None]).to(torch.float8_e4m3fn), scale


def _rows(g, *shape):
    """Activations: channels of different spread, as projections of a trained model give them."""
    spread = torch.exp(0.5 * torch.randn(shape[-1], generator=g, device="cuda"))
    return torch.randn(*shape, generator=g, device="cuda") * (spread / spread.square().mean().sqrt())


def _pages(g, case, lengths):
    """Page pools of keys and values (filled), scales (8 bits), and a table of scattered pages."""
    page, hkv, dim = case["page"], case["heads_kv"], case["head_dim"]
    need = [-(-n // page) for n in lengths]
    total = sum(need) + 3
    order = torch.randperm(total, generator=g, device="cuda").to(torch.int32)
    table = torch.full((len(lengths), max(need)), -1, dtype=torch.int32, device="cuda")
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    pools, scales = [], []
    for _ in range(2):
        x = _rows(g, total, page, hkv, dim)
        if case["cache"] == "fp8":
            x, s = _quantise(x)
            scales.append(s)
        pools.append(x.to(DTYPES[case["cache"]]))
    return pools[0], pools[1], (scales or [None, None])[0], (scales or [None, None])[1], table


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    dt = DTYPES[case["dtype"]]
    st = {"case": case}
    if case["op"] == "rotary":
        sides, hq, hkv, dim = _sides(case), case["heads"], case["heads_kv"], case["head_dim"]
        fused = _rows(g, case["batch"], *sides, hq + 2 * hkv, dim).to(dt)
        st["query"], st["key"], _ = fused.split((hq, hkv, hkv), dim=-2)
        st["positions"] = None
        if case["explicit"]:
            st["positions"] = torch.randint(0, 32768, (case["batch"], *sides, len(sides)), generator=g,
                                            device="cuda", dtype=torch.int32)
        if case["train"]:
            st["query"], st["key"] = (st[n].contiguous().requires_grad_() for n in ("query", "key"))
            st["d_query"] = torch.randn(st["query"].shape, generator=g, device="cuda").to(dt)
            st["d_key"] = torch.randn(st["key"].shape, generator=g, device="cuda").to(dt)
        return st
    lengths = _lengths(case)
    order = torch.randperm(len(lengths), generator=g, device="cuda")
    lengths = [lengths[i] for i in order.tolist()]
    (st["key_pages"], st["value_pages"], st["key_scales"], st["value_scales"],
     st["table"]) = _pages(g, case, lengths)
    st["lengths"] = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    hkv, dim, batch = case["heads_kv"], case["head_dim"], case["batch"]
    if case["op"] == "decode":
        st["query"] = (1.5 * _rows(g, batch, case["new"], case["heads"], dim)).to(dt)
    if case["op"] == "write":
        # the last tokens of each sequence: as many as the call gives, or all where it has fewer
        st["counts"] = st["lengths"].clamp_max(case["new"])
        st["start"] = st["lengths"] - st["counts"]
        fused = _rows(g, batch, case["new"], 2 * hkv, dim).to(dt)
        st["key"], st["value"] = fused.split(hkv, dim=-2)
    return st


# ---- the plain forms ---------------------------------------------------------------------------------

def _gather(pages, scales, page, slot):
    x = pages[page, slot].float()
    return x if scales is None else x * scales[page, slot][..., None]


def _plain_decode(st):
    case, q, table, lengths = st["case"], st["query"], st["table"], st["lengths"]
    B, T, Hq, D = q.shape
    hkv, ps, d = case["heads_kv"], case["page"], case["dilation"]
    K = min(case["kernel"] or case["high"], case["high"])
    at = lengths[:, None].long() - T + torch.arange(T, device=q.device)               # [B, T]
    j = at[..., None] - d * torch.arange(K, device=q.device)                          # [B, T, K]
    valid = j >= 0
    j = j.clamp_min(0)
    page = torch.gather(table.long(), 1, (j // ps).flatten(1)).view_as(j)
    k = _gather(st["key_pages"], st["key_scales"], page, j % ps)
    v = _gather(st["value_pages"], st["value_scales"], page, j % ps)
    logits = torch.einsum("bthgd,btkhd->bthgk", q.float().view(B, T, hkv, Hq // hkv, D), k) * D ** -0.5
    logits = logits.masked_fill(~valid[:, :, None, None, :], -math.inf)
    top = logits.amax(-1, keepdim=True)
    p = torch.exp(logits - torch.where(top == -math.inf, 0.0, top))
    s = p.sum(-1, keepdim=True)
    out = torch.einsum("bthgk,btkhd->bthgd", p, v) / torch.where(s == 0, 1.0, s)
    return {"out": out.reshape(B, T, Hq, D).to(q.dtype), "lse": (top + s.log()).reshape(B, T, Hq)}


def _plain_write(st):
    case, key = st["case"], st["key"]
    B, T = key.shape[:2]
    # a token behind a sequence's own is written as the sequence's last one once more
    t = torch.minimum(torch.arange(T, device=key.device)[None], st["counts"][:, None].long() - 1)
    j = st["start"][:, None].long() + t
    page, slot = torch.gather(st["table"].long(), 1, j // case["page"]), j % case["page"]
    for x, pages, scales in ((key, st["key_pages"], st["key_scales"]),
                             (st["value"], st["value_pages"], st["value_scales"])):
        x = x[torch.arange(B, device=x.device)[:, None], t]
        if scales is not None:
            x, s = _quantise(x.float())
            scales[page, slot] = s
            pages.view(torch.uint8)[page, slot] = x.view(torch.uint8)
        else:
            pages[page, slot] = x


def _plain_read(st):
    case, lengths = st["case"], st["lengths"]
    j = torch.arange(case["high"], device=lengths.device)[None].expand(case["batch"], -1)
    valid = j < lengths[:, None]
    j = torch.where(valid, j, 0)
    page = torch.gather(st["table"].long(), 1, j // case["page"])
    out = []
    for n in ("key", "value"):
        x = _gather(st[n + "_pages"], st[n + "_scales"], page, j % case["page"])
        out.append(x.masked_fill(~valid[..., None, None], 0.0).to(DTYPES[case["dtype"]]))
    return out


def _axis_dims(dim, axes):
    """Channels of each axis: equal parts in steps of 8, the first axes taking what is left over."""
    return [8 * (dim // 8 // axes + (a < dim // 8 % axes)) for a in range(axes)]


def _angles(st, axes, sides, device):
    """One angle for each token and pair of channels, axis after axis, in 64 bits."""
    out = []
    for a, dim in enumerate(_axis_dims(st["case"]["head_dim"], axes)):
        freq = 10000.0 ** (-torch.arange(0, dim, 2, device=device, dtype=torch.float64) / dim)
        if st["positions"] is not None:
            at = st["positions"][..., a].double()
        else:
            at = torch.arange(sides[a], device=device, dtype=torch.float64)
            at = at.view([1] + [-1 if i == a else 1 for i in range(axes)]).expand(1, *sides)
        out.append(at[..., None] * freq)
    return out


def _turn(x, angles, interleaved):
    parts, at = [], 0
    for ang in angles:
        c, s = ang.cos().float().unsqueeze(-2), ang.sin().float().unsqueeze(-2)
        n = 2 * ang.shape[-1]
        y = x[..., at:at + n].float()
        if interleaved:
            u, w = y[..., 0::2], y[..., 1::2]
            parts.append(torch.stack((u * c - w * s, u * s + w * c), -1).flatten(-2))
        else:
            u, w = y.chunk(2, -1)
            parts += [u * c - w * s, u * s + w * c]
        at += n
    return torch.cat(parts, -1).to(x.dtype)


def _plain_rotary(st):
    q, k = st["query"], st["key"]
    sides = q.shape[1:-2]
    angles = _angles(st, len(sides), sides, q.device)
    return _turn(q, angles, st["case"]["interleaved"]), _turn(k, angles, st["case"]["interleaved"])


# ---- one pass ----------------------------------------------------------------------------------------

def run(state):
    st, case = state, state["case"]
    if own:
        import natten_b200 as nb
    if case["op"] == "rotary":
        if own:
            q, k = nb.rotary(st["query"], st["key"], positions=st["positions"],
                             interleaved=case["interleaved"])
        else:
            q, k = _plain_rotary(st)
        if not case["train"]:
            return {"query": q, "key": k}
        dq, dk = torch.autograd.grad((q, k), (st["query"], st["key"]), (st["d_query"], st["d_key"]))
        return {"query": q.detach(), "key": k.detach(), "d_query": dq, "d_key": dk}
    if own:
        cache = nb.KVCache(st["key_pages"], st["value_pages"], st["key_scales"], st["value_scales"])
    if case["op"] == "decode":
        if not own:
            return _plain_decode(st)
        out, lse = nb.na1d_decode(st["query"], cache, st["table"], st["lengths"],
                                  kernel_size=case["kernel"] or None, dilation=case["dilation"],
                                  return_lse=True)
        return {"out": out, "lse": lse}
    if case["op"] == "write":
        if own:
            nb.kv_cache_write(cache, st["key"], st["value"], st["table"], st["start"], st["counts"])
        else:
            _plain_write(st)
        return {n: st[n] for n in ("key_pages", "value_pages", "key_scales", "value_scales")}
    if own:
        key, value = nb.kv_cache_read(cache, st["table"], case["high"], counts=st["lengths"],
                                      dtype=DTYPES[case["dtype"]])
    else:
        key, value = _plain_read(st)
    return {"key": key, "value": value}


def work(case):
    b = BYTES[case["dtype"]]
    if case["op"] == "rotary":
        n = case["batch"] * math.prod(_sides(case)) * (case["heads"] + case["heads_kv"]) * case["head_dim"]
        passes = 2 if case["train"] else 1
        at = 4 * case["batch"] * math.prod(_sides(case)) * len(_sides(case)) if case["explicit"] else 0
        return {"bytes": passes * (2 * n * b + at), "flops": passes * 3 * n}
    row = case["head_dim"] * BYTES[case["cache"]] + (4 if case["cache"] == "fp8" else 0)
    hkv, dim, lengths = case["heads_kv"], case["head_dim"], _lengths(case)
    if case["op"] == "decode":
        d, T = case["dilation"], case["new"]
        met = [0, 0]      # (key, query token) pairs; different keys that a sequence's queries attend
        for n in lengths:
            pairs = [min(case["kernel"] or p + 1, p // d + 1) for p in range(max(0, n - T), n)]
            met[0] += sum(pairs)
            first = max(0, n - T)
            if d == 1:
                met[1] += n - (first + 1 - pairs[0])
            else:
                met[1] += sum(pairs) if T <= d else min(sum(pairs), n)
        io = case["batch"] * T * case["heads"] * (2 * dim * b + 4)
        return {"bytes": 2 * met[1] * hkv * row + io, "flops": 4 * met[0] * case["heads"] * dim}
    if case["op"] == "write":
        n = sum(min(x, case["new"]) for x in lengths) * hkv
        return {"bytes": 2 * n * (dim * b + row), "flops": (4 if case["cache"] == "fp8" else 0) * n * dim}
    n = sum(lengths) * hkv
    return {"bytes": 2 * (n * row + case["batch"] * case["high"] * hkv * dim * b),
            "flops": (2 if case["cache"] == "fp8" else 0) * n * dim}


# ---- the definitions in 64 bits ------------------------------------------------------------------------

def _exact_rows(st, name, b, positions):
    ps = st["case"]["page"]
    page = st["table"][b].long()[positions // ps]
    rows = st[name + "_pages"][page, positions % ps].double()
    if st[name + "_scales"] is not None:
        rows = rows * st[name + "_scales"][page, positions % ps].double().unsqueeze(-1)
    return rows                                                        # [n, Hkv, D]


def _exact_decode(st):
    case, q = st["case"], st["query"].double()
    B, T, Hq, D = q.shape
    group = Hq // case["heads_kv"]
    out = torch.zeros_like(q)
    lse = torch.full((B, T, Hq), -math.inf, dtype=torch.float64, device=q.device)
    for b, n in enumerate(st["lengths"].tolist()):
        for t in range(T):
            p = n - T + t
            if p < 0:
                continue
            first = p % case["dilation"]
            if case["kernel"]:
                first = max(first, p - (case["kernel"] - 1) * case["dilation"])
            at = torch.arange(first, p + 1, case["dilation"], device=q.device)
            k = _exact_rows(st, "key", b, at).repeat_interleave(group, dim=1)
            v = _exact_rows(st, "value", b, at).repeat_interleave(group, dim=1)
            logits = (q[b, t][None] * k).sum(-1) / math.sqrt(D)        # [n, Hq]
            lse[b, t] = torch.logsumexp(logits, 0)
            out[b, t] = (torch.softmax(logits, 0).unsqueeze(-1) * v).sum(0)
    return {"out": out, "lse": lse}


def _exact_write(st):
    case, got = st["case"], {}
    for n in ("key", "value"):
        pages = st[n + "_pages"].double()
        scales = None if st[n + "_scales"] is None else st[n + "_scales"].double()
        for b in range(case["batch"]):
            count, start = int(st["counts"][b]), int(st["start"][b])
            at = torch.arange(start, start + count, device=pages.device)
            page, slot = st["table"][b].long()[at // case["page"]], at % case["page"]
            x = st[n][b, :count].double()
            if scales is not None:
                s = x.abs().max(-1).values / E4M3_MAX
                s = torch.where(s < SMALLEST_SCALE, SMALLEST_SCALE, s)
                scales[page, slot] = s
                x = x / s.unsqueeze(-1)
            pages[page, slot] = x
        got[n + "_pages"], got[n + "_scales"] = pages, scales
    return got


def _exact_read(st):
    case, got = st["case"], {}
    for n in ("key", "value"):
        x = torch.zeros(case["batch"], case["high"], case["heads_kv"], case["head_dim"],
                        dtype=torch.float64, device="cuda")
        for b, m in enumerate(st["lengths"].tolist()):
            x[b, :m] = _exact_rows(st, n, b, torch.arange(m, device="cuda"))
        got[n] = x
    return got


def _exact_rotary(st):
    """Every pair of channels as a complex number times exp(i angle)."""
    case, sides = st["case"], _sides(st["case"])
    dims = _axis_dims(case["head_dim"], len(sides))

    def turn(x, sign):
        y, at = torch.empty(x.shape, dtype=torch.float64, device=x.device), 0
        for a, dim in enumerate(dims):
            half = dim // 2
            i = torch.arange(half, device=x.device)
            one, two = (at + 2 * i, at + 2 * i + 1) if case["interleaved"] else (at + i, at + half + i)
            if st["positions"] is not None:
                place = st["positions"].select(-1, a).double()
            else:
                place = torch.arange(sides[a], device=x.device).double()
                place = place.reshape([1] + [sides[a] if b == a else 1 for b in range(len(sides))])
            phase = place.unsqueeze(-1) / torch.pow(torch.tensor(1e4, dtype=torch.float64, device=x.device),
                                                    2.0 * i.double() / dim)
            z = torch.complex(x[..., one].double(), x[..., two].double())
            z = z * torch.polar(torch.ones_like(phase), sign * phase).unsqueeze(-2)
            y[..., one], y[..., two] = z.real, z.imag
            at += dim
        return y

    with torch.no_grad():
        got = {"query": turn(st["query"], 1.0), "key": turn(st["key"], 1.0)}
        if case["train"]:
            got["d_query"], got["d_key"] = turn(st["d_query"], -1.0), turn(st["d_key"], -1.0)
    return got


def exact(case, seed):
    st = prepare(case, seed)
    return {"decode": _exact_decode, "write": _exact_write, "read": _exact_read,
            "rotary": _exact_rotary}[case["op"]](st)
