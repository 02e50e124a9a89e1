"""The paged serving path's operators, as measurable cases.

Four kinds of pass, each through the package's public entry points:

* ``rotary``: rotary positions of the queries and keys of a call's tokens
  (``apply_rotary``), half or traditional pairs, the whole head or part of it,
  plain or YaRN frequencies;
* ``cache``: a layer's new keys and values written into the paged cache
  (``PagedKVCache.write``, rotating queries and keys on the way) and read back
  (``PagedKVCache.read``), in 16 or 8 bits; ``fresh=0`` reads a cached prefix;
* ``attention``: ``paged_sdpa`` of new tokens over the paged cache, from one
  decode row to whole prompts, alone, batched and mixed;
* ``layer``: write and attention together, as a decoder layer makes them.

The plain form keeps its pages as ``[page, kv head, slot, dim]`` and computes
in 32 bits; angles in 64.
"""

from __future__ import annotations

import math

import torch

own = False
DEV = "cuda"


def listed():
    return [
        # The rotation of one decoded token: the smallest call.
        dict(name="rotary_token", kind="rotary", t=1, hq=40, hkv=8, d=128, dims=128, trad=False, yarn=1.0, far=4096),
        # A whole prompt's, with positions scaled to eight times the trained length.
        dict(name="rotary_prompt", kind="rotary", t=8192, hq=40, hkv=8, d=128, dims=128, trad=False, yarn=8.0,
             far=262144),
        # A prompt chunk of a decoder that rotates pairs side by side, in half of each head, far out.
        dict(name="rotary_partial", kind="rotary", t=2000, hq=32, hkv=4, d=128, dims=64, trad=True, yarn=1.0,
             far=1000000),
        # One decode step of sixteen requests into 8-bit pages, and the rows it wrote.
        dict(name="cache_decode_8bit", kind="cache", b=16, rows=1, spread=0.0, ctx=8192, hq=40, hkv=8, d=128, bits=8,
             page=64, fresh=1),
        # A prompt into 8-bit pages and back.
        dict(name="cache_prompt_8bit", kind="cache", b=1, rows=8192, spread=0.0, ctx=8192, hq=40, hkv=8, d=128,
             bits=8, page=64, fresh=1),
        # A cached prefix of eight requests read back from 8-bit pages.
        dict(name="cache_prefix_8bit", kind="cache", b=8, rows=1, spread=1.0, ctx=8192, hq=40, hkv=8, d=128, bits=8,
             page=64, fresh=0),
        # One decoded token of one request at 4k.
        dict(name="attention_token", kind="attention", b=1, rows=1, spread=0.0, ctx=4096, hq=40, hkv=8, d=128,
             bits=16, page=64),
        # The verify rows of sixteen requests of very different lengths up to 32k, 8-bit pages.
        dict(name="attention_verify_8bit", kind="attention", b=16, rows=4, spread=1.0, ctx=32768, hq=40, hkv=8, d=128,
             bits=8, page=64),
        # A chunk of a long prompt.
        dict(name="attention_chunk", kind="attention", b=1, rows=512, spread=0.0, ctx=16384, hq=40, hkv=8, d=128,
             bits=16, page=64),
        # Whole prompts of different lengths, packed.
        dict(name="attention_prompts", kind="attention", b=4, rows=4096, spread=1.0, ctx=4096, hq=40, hkv=8, d=128,
             bits=16, page=64),
        # A prompt chunk beside fifteen decoding requests, 8-bit pages.
        dict(name="attention_mixed_8bit", kind="attention", b=16, rows=1000, spread=-1.0, ctx=8192, hq=32, hkv=4,
             d=128, bits=8, page=128),
        # One decoder layer's cache work for a chunk: rotate, write, attend.
        dict(name="layer_chunk", kind="layer", b=2, rows=256, spread=0.5, ctx=8192, hq=40, hkv=8, d=128, bits=16,
             page=64),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["rotary", "cache", "cache", "attention", "attention", "attention", "layer"])
    hq, hkv, d = rng.choice([(40, 8, 128), (40, 8, 128), (32, 4, 128), (16, 2, 128), (8, 8, 128), (16, 4, 64),
                             (24, 4, 256)])
    if kind == "rotary":
        return dict(kind=kind, t=_log(rng, 1, 8192), hq=hq, hkv=hkv, d=d, dims=rng.choice([d, d, d // 2, d // 4]),
                    trad=rng.random() < 0.4, yarn=rng.choice([1.0, 1.0, 4.0, 32.0]), far=_log(rng, 8192, 1000000))
    bits, page = rng.choice([16, 8]), rng.choice([32, 64, 64, 128, 256])
    if kind == "cache":
        b, fresh = _log(rng, 1, 16), rng.choice([1, 1, 0])
        rows = _log(rng, 1, 8192 // b) if fresh else 1
        return dict(kind=kind, b=b, rows=rows, spread=round(rng.random(), 3), ctx=8192 if fresh else _log(rng, 64, 8192),
                    hq=hq, hkv=hkv, d=d, bits=bits, page=page, fresh=fresh)
    shape = rng.choice(["decode", "decode", "chunk", "prompts", "mixed"]) if kind == "attention" else "chunk"
    if shape == "decode":
        return dict(kind=kind, b=_log(rng, 1, 16), rows=rng.randint(1, 8), spread=round(rng.random(), 3),
                    ctx=_log(rng, 64, 32768), hq=hq, hkv=hkv, d=d, bits=bits, page=page)
    if shape == "chunk":
        rows = _log(rng, 8, 512)
        return dict(kind=kind, b=rng.randint(1, 2), rows=rows, spread=round(rng.random(), 3),
                    ctx=_log(rng, rows + 1, 16384), hq=hq, hkv=hkv, d=d, bits=bits, page=page)
    if shape == "prompts":
        rows = _log(rng, 16, 4096 if d < 256 else 3600)
        return dict(kind=kind, b=rng.randint(1, 4), rows=rows, spread=round(rng.random(), 3), ctx=rows, hq=hq,
                    hkv=hkv, d=d, bits=bits, page=page)
    rows = _log(rng, 16, 1000)
    return dict(kind=kind, b=rng.randint(2, 16), rows=rows, spread=-1.0, ctx=_log(rng, rows + 1, 8192), hq=hq,
                hkv=hkv, d=d, bits=bits, page=page)


# -- inputs ---------------------------------------------------------------------

def _shape(c):
    """(new tokens, context after them) of each request: the first has rows and
    ctx, the others spread evenly below them; spread -1: the others decode one token."""
    rows, ctx = [c["rows"]], [c["ctx"]]
    for i in range(1, c["b"]):
        u, w = 0.6180339887 * i % 1.0, 0.4142135624 * i % 1.0
        if c["spread"] < 0:
            rows.append(1)
            ctx.append(max(1, int(c["ctx"] * (0.06 + 0.94 * u))))
            continue
        rows.append(max(1, int(c["rows"] * (1.0 - 0.8 * c["spread"] * w))))
        if c["rows"] == c["ctx"]:
            ctx.append(rows[-1])   # prompts from their first token
        else:
            ctx.append(max(rows[-1], int(c["ctx"] * (1.0 - 0.95 * c["spread"] * u))))
    return rows, ctx


def _randn(gen, *shape):
    return torch.randn(shape, device=DEV, generator=gen).to(torch.bfloat16)


def _rows(gen, t, h, d):
    """Projected rows of a decoder: a few channels of each head much larger."""
    x = torch.randn((t, h, d), device=DEV, generator=gen)
    x *= torch.exp(0.5 * torch.randn((1, h, d), device=DEV, generator=gen))
    return x.to(torch.bfloat16)


def _quantised(x):
    """(values of 8 bits, one 32-bit scale per row) of rows in their last dimension."""
    top = x.float().abs().amax(-1)
    q = torch.round(x.float() * (127.0 / top).unsqueeze(-1))
    return q.to(torch.int8), top / 127.0


def _inv_freq(dims, yarn, base=1.0e6, trained=32768, fast=32.0, slow=1.0):
    """(float64 radians per position of each pair, factor of the rotated values)."""
    f = base ** (-torch.arange(0, dims, 2, dtype=torch.float64) / dims)
    if yarn <= 1.0:
        return f, 1.0
    edge = [dims * math.log(trained / (n * 2.0 * math.pi)) / (2.0 * math.log(base)) for n in (fast, slow)]
    lo, hi = max(math.floor(edge[0]), 0), min(math.ceil(edge[1]), dims - 1)
    ramp = ((torch.arange(dims // 2, dtype=torch.float64) - lo) / max(hi - lo, 0.001)).clamp(0.0, 1.0)
    return f * (1.0 - ramp) + f / yarn * ramp, 0.1 * math.log(yarn) + 1.0


def _table(c):
    """The framework's rotary plan of a case."""
    from mtplx_amd.rotary import rotary_table

    dims, trad, yarn = c.get("dims", c["d"]), c.get("trad", False), c.get("yarn", 1.0)
    more = dict(scaling="yarn", factor=yarn, trained_positions=32768) if yarn > 1.0 else {}
    return rotary_table(dims, base=1.0e6, traditional=trad, device=DEV, **more)


def _rotary_inputs(c, seed):
    gen = torch.Generator(device=DEV).manual_seed(int(seed))
    q, k = _rows(gen, c["t"], c["hq"], c["d"]), _rows(gen, c["t"], c["hkv"], c["d"])
    first = torch.randint(0, max(1, c["far"] - c["t"]), (1,), device=DEV, generator=gen)
    return q, k, (first + torch.arange(c["t"], device=DEV)).to(torch.int32)


def _paged_inputs(c, seed):
    gen = torch.Generator(device=DEV).manual_seed(int(seed))
    rows, ctx = _shape(c)
    page, hkv, d, t = c["page"], c["hkv"], c["d"], sum(rows)
    width = max(-(-n // page) for n in ctx)
    pages = sum(-(-n // page) for n in ctx) + 2
    # Pages of a pool that other requests have used: any order.
    order = torch.randperm(pages, device=DEV, generator=gen).to(torch.int32)
    table = torch.full((c["b"], width), -1, dtype=torch.int32, device=DEV)
    at = 0
    for b, n in enumerate(ctx):
        used = -(-n // page)
        table[b, :used] = order[at:at + used]
        at += used
    s = dict(table=table, pages=pages, rows=rows, ctx=ctx, max_rows=max(rows), t=t)
    s["row_off"] = torch.tensor([sum(rows[:i]) for i in range(len(rows) + 1)], dtype=torch.int32, device=DEV)
    s["start"] = torch.tensor([n - r for n, r in zip(ctx, rows)], dtype=torch.int32, device=DEV)
    s["q"] = _rows(gen, t, c["hq"], d)
    s["k"], s["v"] = _rows(gen, t, hkv, d), _rows(gen, t, hkv, d)
    # What the pages hold: rows of unit size, keys as they are after rotation.
    s["old"] = [_randn(gen, pages, hkv, page, d) for _ in range(2)]
    return s


def prepare(case, seed):
    c = dict(case)
    if c["kind"] == "rotary":
        q, k, pos = _rotary_inputs(c, seed)
        s = dict(c=c, q=q, k=k, pos=pos)
        if own:
            s["rotary"] = _table(c)
        else:
            s["freq"], s["gain"] = _inv_freq(c["dims"], c["yarn"])
            s["freq"] = s["freq"].to(DEV)
        return s
    s = _paged_inputs(c, seed)
    s["c"] = c
    old = s.pop("old")
    if own:
        from mtplx_amd.paged_kv_cache import PagedKVCache

        cache = PagedKVCache(s["pages"], c["hkv"], c["d"], page_size=c["page"], bits=c["bits"], device=DEV)
        every = torch.arange(s["pages"], dtype=torch.int32, device=DEV).unsqueeze(1)
        cache.write(*(x.transpose(1, 2).reshape(-1, c["hkv"], c["d"]) for x in old), every,
                    torch.zeros(s["pages"], dtype=torch.int32, device=DEV))
        s["cache"], s["rotary"] = cache, _table(c)
    else:
        s["freq"] = _inv_freq(c["d"], 1.0)[0].to(DEV)
        if c["bits"] == 8:
            s["pool"] = [_quantised(x) for x in old]
        else:
            s["pool"] = old
    return s


# -- the plain form -------------------------------------------------------------

def _rotated(x, angle, dims, trad, gain):
    """Rows [T, H, D] in float32 rotated by angle [T, dims / 2] (float64), rounded once."""
    cs, sn = (gain * angle.cos()).float().unsqueeze(1), (gain * angle.sin()).float().unsqueeze(1)
    r = x[..., :dims].float()
    x1, x2 = (r[..., 0::2], r[..., 1::2]) if trad else (r[..., :dims // 2], r[..., dims // 2:])
    y1, y2 = x1 * cs - x2 * sn, x1 * sn + x2 * cs
    y = torch.stack([y1, y2], dim=-1).flatten(-2) if trad else torch.cat([y1, y2], dim=-1)
    return torch.cat([y.to(x.dtype), x[..., dims:]], dim=-1)


def _token_places(s):
    """(request, index in it, position) of each new token."""
    at = torch.arange(s["t"], device=DEV)
    b = torch.searchsorted(s["row_off"][1:].long(), at, right=True)
    i = at - s["row_off"].long()[b]
    return b, i, s["start"].long()[b] + i


def _plain_write(s):
    """The new rows into the pages; returns the rotated queries."""
    c = s["c"]
    b, _, pos = _token_places(s)
    angle = pos.double().unsqueeze(1) * s["freq"]
    q, k = (_rotated(x, angle, c["d"], False, 1.0) for x in (s["q"], s["k"]))
    page, slot = s["table"].long()[b, pos // c["page"]], pos % c["page"]
    for pool, x in zip(s["pool"], (k, s["v"])):
        if c["bits"] == 8:
            for part, value in zip(pool, _quantised(x)):
                part[page, :, slot] = value
        else:
            pool[page, :, slot] = x
    return q


def _plain_pages(s, pool):
    """float32 [B, Hkv, keys, D] that a request's pages hold (absent pages: page 0, masked later)."""
    at = s["table"].long().clamp(min=0)
    if s["c"]["bits"] == 8:
        x = pool[0][at].float() * pool[1][at].unsqueeze(-1)
    else:
        x = pool[at].float()
    return x.transpose(1, 2).flatten(2, 3)


def _plain_read(s, start, count, lengths):
    """bf16 [B, Hkv, count, D] of the positions from start on, zeros from lengths on."""
    b = torch.arange(s["table"].shape[0], device=DEV)
    pos = start.long().unsqueeze(1) + torch.arange(count, device=DEV)
    live = pos < lengths.long().unsqueeze(1)
    pos = torch.where(live, pos, torch.zeros_like(pos))
    page, slot = s["table"].long()[b.unsqueeze(1), pos // s["c"]["page"]], pos % s["c"]["page"]
    got = []
    for pool in s["pool"]:
        x = pool[0][page, :, slot].float() * pool[1][page, :, slot].unsqueeze(-1) if s["c"]["bits"] == 8 \
            else pool[page, :, slot].float()
        got.append((x * live[..., None, None]).to(torch.bfloat16).transpose(1, 2).contiguous())
    return tuple(got)


def _plain_attention(s, q):
    c = s["c"]
    hq, hkv, d = c["hq"], c["hkv"], c["d"]
    rep, top = hq // hkv, s["max_rows"]
    k, v = (_plain_pages(s, pool) for pool in s["pool"])
    at = (s["row_off"][:-1].long().unsqueeze(1) + torch.arange(top, device=DEV)).clamp(max=s["t"] - 1)
    qp = q.float()[at].reshape(c["b"], top, hkv, rep, d).permute(0, 2, 3, 1, 4).reshape(c["b"], hkv, rep * top, d)
    score = torch.matmul(qp * (1.0 / math.sqrt(d)), k.transpose(2, 3).contiguous()).view(c["b"], hkv, rep, top, -1)
    pos = s["start"].long().unsqueeze(1) + torch.arange(top, device=DEV)
    hidden = torch.arange(k.shape[2], device=DEV) > pos.unsqueeze(-1)
    score = score.masked_fill_(hidden[:, None, None], float("-inf"))
    score -= score.amax(-1, keepdim=True)
    score = score.exp_()
    total = score.sum(-1, keepdim=True)
    o = torch.matmul(score.view(c["b"], hkv, rep * top, -1), v).view(c["b"], hkv, rep, top, d) / total
    b, i, _ = _token_places(s)
    return o.permute(0, 3, 1, 2, 4).reshape(c["b"], top, hq, d)[b, i].to(torch.bfloat16)


# -- one pass -------------------------------------------------------------------

def _read_range(s):
    """What the read half of a cache pass asks for: the new rows, or the cached prefix."""
    if s["c"]["fresh"]:
        return s["start"], s["max_rows"], s["start"] + (s["row_off"][1:] - s["row_off"][:-1])
    return torch.zeros_like(s["start"]), s["c"]["ctx"] - s["c"]["rows"], s["start"]


def _write(s):
    if not own:
        return _plain_write(s)
    return s["cache"].write(s["k"], s["v"], s["table"], s["start"], s["row_off"], max_rows=s["max_rows"],
                            queries=s["q"], rotary=s["rotary"])


def _attention(s, q):
    if not own:
        return _plain_attention(s, q)
    from mtplx_amd.paged_attention import paged_sdpa

    return paged_sdpa(q, s["cache"], s["table"], s["start"], s["row_off"], max_rows=s["max_rows"])


def run(state):
    s = state
    c = s["c"]
    if c["kind"] == "rotary":
        if own:
            from mtplx_amd.rotary import apply_rotary

            return apply_rotary(s["rotary"], s["q"], s["k"], s["pos"])
        angle = s["pos"].double().unsqueeze(1) * s["freq"]
        return tuple(_rotated(x, angle, c["dims"], c["trad"], s["gain"]) for x in (s["q"], s["k"]))
    if c["kind"] == "attention":
        return _attention(s, s["q"])
    if c["kind"] == "layer":
        return _attention(s, _write(s))
    q = _write(s) if c["fresh"] else s["q"]
    start, count, lengths = _read_range(s)
    if own:
        return q, s["cache"].read(s["table"], count, start=start, lengths=lengths)
    return q, _plain_read(s, start, count, lengths)


# -- from the definition, in 64 bits --------------------------------------------

def _exact_rotated(x, pos, dims, trad, yarn):
    freq, gain = _inv_freq(dims, yarn)
    z = torch.polar(torch.full((pos.numel(), dims // 2), gain, dtype=torch.float64, device=DEV),
                    pos.double().unsqueeze(1) * freq.to(DEV)).unsqueeze(1)
    x = x.double()
    first, second = (slice(0, dims, 2), slice(1, dims, 2)) if trad else (slice(0, dims // 2), slice(dims // 2, dims))
    w = torch.complex(x[..., first], x[..., second]) * z
    y = x.clone()
    y[..., first], y[..., second] = w.real, w.imag
    return y


def _exact_stored(x, bits):
    """The values that rows stand for once they are stored (float64 rows in)."""
    x = x.to(torch.bfloat16).double()
    if bits == 16:
        return x
    top = x.abs().amax(-1, keepdim=True)
    return torch.round(x * (127.0 / top.float()).double()) * (top / 127.0)


def exact(case, seed):
    c = dict(case)
    if c["kind"] == "rotary":
        q, k, pos = _rotary_inputs(c, seed)
        return tuple(_exact_rotated(x, pos, c["dims"], c["trad"], c["yarn"]) for x in (q, k))
    s = dict(_paged_inputs(c, seed), c=c)
    d, rep, page = c["d"], c["hq"] // c["hkv"], c["page"]
    writes = c["kind"] == "layer" or (c["kind"] == "cache" and c["fresh"])
    whole, q_all = [], []
    for b, (rows, ctx) in enumerate(zip(s["rows"], s["ctx"])):
        lo = int(s["row_off"][b])
        ids = s["table"][b, :-(-ctx // page)].long()
        kv = [_exact_stored(x[ids].transpose(0, 1).reshape(c["hkv"], -1, d)[:, :ctx].double(), c["bits"])
              for x in s["old"]]
        q = s["q"][lo:lo + rows].double()
        if writes:
            pos = torch.arange(ctx - rows, ctx, device=DEV)
            q = _exact_rotated(s["q"][lo:lo + rows], pos, d, False, 1.0)
            k = _exact_rotated(s["k"][lo:lo + rows], pos, d, False, 1.0)
            for x, new in zip(kv, (k, s["v"][lo:lo + rows].double())):
                x[:, ctx - rows:] = _exact_stored(new, c["bits"]).transpose(0, 1)
        whole.append(kv)
        q_all.append(q)
    if c["kind"] == "cache":
        q = torch.cat(q_all)
        start, count, lengths = _read_range(s)
        got = [torch.zeros((c["b"], c["hkv"], count, d), dtype=torch.float64, device=DEV) for _ in range(2)]
        for b in range(c["b"]):
            lo, hi = int(start[b]), int(lengths[b])
            for x, kv in zip(got, whole[b]):
                x[b, :, :hi - lo] = kv[:, lo:hi]
        return q, tuple(got)
    out = []
    for rows, ctx, (k, v), q in zip(s["rows"], s["ctx"], whole, q_all):
        if writes:
            q = q.to(torch.bfloat16).double()   # what a layer hands from the rotation to the attention
        o = torch.empty((rows, c["hq"], d), dtype=torch.float64, device=DEV)
        hidden = torch.arange(ctx, device=DEV) > torch.arange(ctx - rows, ctx, device=DEV).unsqueeze(1)
        for h in range(c["hq"]):
            score = (q[:, h] @ k[h // rep].T) / math.sqrt(d)
            o[:, h] = torch.softmax(score.masked_fill(hidden, float("-inf")), dim=-1) @ v[h // rep]
        out.append(o)
    return torch.cat(out)


def work(case):
    c = dict(case)
    if c["kind"] == "rotary":
        n = c["t"] * (c["hq"] + c["hkv"]) * c["d"]
        return {"bytes": 4.0 * n + 4.0 * c["t"], "flops": 3.0 * n * c["dims"] / c["d"]}
    rows, ctx = _shape(c)
    t, keys = sum(rows), sum(ctx)
    row = c["hkv"] * (2 * c["d"] if c["bits"] == 16 else c["d"] + 4)   # one stored token of K or V
    made = 4.0 * t * (c["hq"] + c["hkv"]) * c["d"]                     # q in and out, k and v in
    if c["kind"] == "cache":
        if c["fresh"]:
            return {"bytes": made + 4.0 * t * row + 4.0 * t * c["hkv"] * c["d"], "flops": 8.0 * t * c["hq"] * c["d"]}
        n = keys - t
        return {"bytes": 2.0 * n * row + 4.0 * c["b"] * (c["ctx"] - c["rows"]) * c["hkv"] * c["d"],
                "flops": 2.0 * n * c["hkv"] * c["d"]}
    pairs = sum(r * (n - r) + r * (r + 1) / 2.0 for r, n in zip(rows, ctx))
    moved = 2.0 * keys * row + 4.0 * t * c["hq"] * c["d"]
    if c["kind"] == "layer":
        moved += made
    return {"bytes": moved, "flops": 4.0 * pairs * c["hq"] * c["d"]}
