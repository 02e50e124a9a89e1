"""What a decoder layer of the paged serving path does beside the plain causal
form, as measurable cases.

Five kinds of pass, each through the package's public entry points:

* ``positions``: queries and keys of a call's tokens, each head normalised and
  rotated in one pass (``apply_rotary`` with ``norms``), by one position or by
  several axes (a table with ``sections``);
* ``write``: a layer's new keys and values into the paged cache, keys and queries
  normalised and rotated on the way (``PagedKVCache.write`` with ``norms`` and
  ``positions``), and what was stored read back;
* ``window``: ``paged_sdpa`` with a sliding window and first tokens that stay
  visible; pages that no new token sees have been given back;
* ``prefix``: ``paged_sdpa`` of a batch whose requests share their first pages;
* ``layer``: write and window together, as a decoder layer makes them.

The plain form keeps its pages as ``[page, kv head, slot, dim]`` and computes
in 32 bits; angles in 64.
"""

from __future__ import annotations

import math

import torch

own = False
DEV = "cuda"
EPS = 1.0e-6


def listed():
    return [
        # One decoded token's heads, normalised and rotated: the smallest call.
        dict(name="norms_token", kind="positions", t=1, hq=40, hkv=8, d=128, dims=128, trad=False, axes=1, turn=False,
             norms=True, far=32768),
        # A whole prompt's.
        dict(name="norms_prompt", kind="positions", t=8192, hq=40, hkv=8, d=128, dims=128, trad=False, axes=1,
             turn=False, norms=True, far=32768),
        # A prompt with a large image: three axes in runs of pairs, no norms.
        dict(name="axes_image", kind="positions", t=8192, hq=32, hkv=4, d=128, dims=128, trad=False, axes=3,
             turn=False, norms=False, far=32768),
        # A chunk of one, axes dealt in turn over a quarter of wide heads, normalised.
        dict(name="axes_norms_partial", kind="positions", t=2000, hq=24, hkv=4, d=256, dims=64, trad=False, axes=3,
             turn=True, norms=True, far=262144),
        # The verify rows of sixteen requests into 8-bit pages, and what was stored.
        dict(name="write_verify_8bit", kind="write", b=16, rows=4, spread=0.0, ctx=8192, hq=40, hkv=8, d=128, bits=8,
             page=64, axes=1, norms=True),
        # A prompt with images into 16-bit pages and back.
        dict(name="write_prompt", kind="write", b=1, rows=8192, spread=0.0, ctx=8192, hq=40, hkv=8, d=128, bits=16,
             page=64, axes=3, norms=True),
        # One decoded token of one long request behind a window.
        dict(name="window_token", kind="window", b=1, rows=1, spread=0.0, ctx=32768, hq=40, hkv=8, d=128, bits=16,
             page=64, window=4096, sinks=4),
        # The verify rows of sixteen requests of very different lengths, 8-bit pages.
        dict(name="window_verify_8bit", kind="window", b=16, rows=4, spread=1.0, ctx=32768, hq=40, hkv=8, d=128,
             bits=8, page=64, window=4096, sinks=64),
        # A whole prompt in a layer that sees the last 1024 tokens.
        dict(name="window_prompt", kind="window", b=1, rows=8192, spread=0.0, ctx=8192, hq=40, hkv=8, d=128, bits=16,
             page=64, window=1024, sinks=0),
        # One decode step of sixteen conversations behind one instruction text.
        dict(name="prefix_decode", kind="prefix", b=16, rows=1, spread=0.8, prefix=8192, tail=600, hq=40, hkv=8, d=128,
             bits=16, page=64),
        # The verify rows of 32 requests about one long document, 8-bit pages.
        dict(name="prefix_verify_8bit", kind="prefix", b=32, rows=4, spread=0.8, prefix=32768, tail=2048, hq=40, hkv=8,
             d=128, bits=8, page=64),
        # One windowed decoder layer's cache work for a chunk: normalise, rotate, write, attend.
        dict(name="layer_window", kind="layer", b=2, rows=256, spread=0.5, ctx=8192, hq=40, hkv=8, d=128, bits=16,
             page=64, window=2048, sinks=4, axes=3, norms=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["positions", "positions", "write", "window", "window", "prefix", "prefix", "layer"])
    hq, hkv, d = rng.choice([(40, 8, 128), (40, 8, 128), (32, 4, 128), (16, 2, 128), (8, 8, 128), (16, 4, 64),
                             (24, 4, 256)])
    if kind == "positions":
        if rng.random() < 0.15:
            hq, hkv, d = 12, 12, 80
        axes = rng.choice([1, 2, 3, 3])
        return dict(kind=kind, t=_log(rng, 1, 8192 if d < 256 else 6000), hq=hq, hkv=hkv, d=d,
                    dims=rng.choice([d, d, d // 2, d // 4]) // 4 * 4, trad=rng.random() < 0.3, axes=axes,
                    turn=rng.random() < 0.5, norms=axes == 1 or rng.random() < 0.6, far=_log(rng, 8192, 1000000))
    bits, page = rng.choice([16, 8]), rng.choice([32, 64, 64, 128, 256])
    spread = round(rng.random(), 3)
    if kind == "write":
        b = _log(rng, 1, 16)
        return dict(kind=kind, b=b, rows=_log(rng, 1, (8192 if d < 256 else 6000) // b), spread=spread, ctx=8192, hq=hq, hkv=hkv, d=d,
                    bits=bits, page=page, axes=rng.choice([1, 3]), norms=rng.random() < 0.8)
    if kind == "prefix":
        return dict(kind=kind, b=_log(rng, 2, 32), rows=rng.randint(1, 4), spread=spread, prefix=_log(rng, 512, 32768),
                    tail=_log(rng, 8, 2048), hq=hq, hkv=hkv, d=d if d < 256 else 128, bits=bits, page=page)
    more = dict(window=_log(rng, 100, 4096), sinks=rng.choice([0, 0, 1, 4, 64, 100]))
    if kind == "layer":
        more.update(axes=rng.choice([1, 3]), norms=rng.random() < 0.8)
    shape = rng.choice(["decode", "decode", "chunk", "prompts"]) if kind == "window" else "chunk"
    if shape == "decode":
        return dict(kind=kind, b=_log(rng, 1, 16), rows=rng.randint(1, 8), spread=spread, ctx=_log(rng, 64, 32768),
                    hq=hq, hkv=hkv, d=d, bits=bits, page=page, **more)
    if shape == "chunk":
        rows = _log(rng, 8, 512)
        return dict(kind=kind, b=rng.randint(1, 2), rows=rows, spread=spread, ctx=_log(rng, rows + 1, 16384), hq=hq,
                    hkv=hkv, d=d, bits=bits, page=page, **more)
    b, more["window"] = rng.randint(1, 4), _log(rng, 100, 1024)
    rows = _log(rng, 16, 8192 // b if d < 256 else 4000 // b)
    return dict(kind=kind, b=b, rows=rows, spread=spread, ctx=rows, hq=hq, hkv=hkv, d=d, bits=bits, page=page, **more)


# -- inputs ---------------------------------------------------------------------

def _shape(c):
    """(new tokens, context after them) of each request: the first has the most,
    the others spread evenly below."""
    top = c["prefix"] + max(c["tail"], c["rows"]) if c["kind"] == "prefix" else c["ctx"]
    rows, ctx = [c["rows"]], [top]
    for i in range(1, c["b"]):
        u, w = 0.6180339887 * i % 1.0, 0.4142135624 * i % 1.0
        if c["kind"] == "prefix":   # every request has its own tail
            rows.append(max(1, int(c["rows"] * (1.0 - 0.8 * c["spread"] * w))))
            ctx.append(c["prefix"] + max(rows[-1], int(c["tail"] * (1.0 - 0.95 * c["spread"] * u))))
            continue
        rows.append(max(1, int(c["rows"] * (1.0 - 0.8 * c["spread"] * w))))
        if c["rows"] == c["ctx"]:
            ctx.append(rows[-1])   # prompts from their first token
        else:
            ctx.append(max(rows[-1], int(c["ctx"] * (1.0 - 0.95 * c["spread"] * u))))
    return rows, ctx


def _rows(gen, t, h, d):
    """Projected rows of a decoder: a few channels of each head much larger."""
    x = torch.randn((t, h, d), device=DEV, generator=gen)
    x *= torch.exp(0.5 * torch.randn((1, h, d), device=DEV, generator=gen))
    return x.to(torch.bfloat16)


def _weight(gen, d):
    """A head norm's weight as models learn it: positive, a few channels far from one."""
    return torch.exp(0.4 * torch.randn(d, device=DEV, generator=gen)).to(torch.bfloat16)


def _axis_positions(first, n, axes):
    """int32 [axes, n] positions of n tokens from `first` on: text, an image in
    the middle half (its time stands still, rows and columns count), text."""
    at = torch.arange(n, device=DEV)
    lo, hi = n // 4, n - n // 4
    side = max(1, math.isqrt(max(0, hi - lo)))
    inside = (at >= lo) & (at < hi)
    grid = [torch.full_like(at, lo), lo + (at - lo) // side, lo + (at - lo) % side]
    return torch.stack([first + torch.where(inside, grid[a], at) for a in range(axes)]).to(torch.int32)


def _quantised(x):
    """(values of 8 bits, one 32-bit scale per row) of rows in their last dimension."""
    top = x.float().abs().amax(-1)
    q = torch.round(x.float() * (127.0 / top).unsqueeze(-1))
    return q.to(torch.int8), top / 127.0


def _frequencies(dims, base=1.0e6):
    """float64 radians per position of each pair."""
    return base ** (-torch.arange(0, dims, 2, dtype=torch.float64) / dims)


def _sections(c):
    """Pairs of each axis (None: one axis), and whether they are dealt in turn."""
    pairs, axes, turn = c.get("dims", c["d"]) // 2, c["axes"], c.get("turn", False)
    if axes == 1:
        return None, False
    side = max(1, pairs * 5 // 16 if turn else pairs * 3 // 8)
    return (pairs - (axes - 1) * side,) + (side,) * (axes - 1), turn


def _axis_of(c):
    """int64 [pairs]: the axis that each pair turns by."""
    sections, turn = _sections(c)
    pairs = c.get("dims", c["d"]) // 2
    i = torch.arange(pairs, device=DEV)
    if sections is None:
        return torch.zeros_like(i)
    if not turn:
        return torch.repeat_interleave(torch.arange(len(sections), device=DEV),
                                       torch.tensor(sections, device=DEV))
    a = i % len(sections)
    return torch.where(i < len(sections) * torch.tensor(sections, device=DEV)[a], a, 0)


def _table(c):
    """The framework's rotary plan of a case."""
    from mtplx_amd.rotary import rotary_table

    sections, turn = _sections(c)
    return rotary_table(c.get("dims", c["d"]), base=1.0e6, traditional=c.get("trad", False), sections=sections,
                        interleaved=turn, device=DEV)


def _positions_inputs(c, seed):
    gen = torch.Generator(device=DEV).manual_seed(int(seed))
    q, k = _rows(gen, c["t"], c["hq"], c["d"]), _rows(gen, c["t"], c["hkv"], c["d"])
    first = torch.randint(0, max(1, c["far"] - c["t"]), (1,), device=DEV, generator=gen)
    pos = _axis_positions(first, c["t"], c["axes"])
    s = dict(c=c, q=q, k=k, pos=pos[0] if c["axes"] == 1 else pos)
    s["wq"], s["wk"] = _weight(gen, c["d"]), _weight(gen, c["d"])
    return s


def _seen_from(c, rows, ctx):
    """First position behind the sinks that a request's new tokens see."""
    if "window" not in c:
        return 0
    return max(0, min(ctx, ctx - rows - c["window"] + 1))


def _paged_inputs(c, seed):
    gen = torch.Generator(device=DEV).manual_seed(int(seed))
    rows, ctx = _shape(c)
    page, hkv, d, t = c["page"], c["hkv"], c["d"], sum(rows)
    width = max(-(-n // page) for n in ctx)
    shared = c.get("prefix", 0) // page   # pages that all requests have in common
    kept = []                             # each request's own pages (the window's others were given back)
    for r, n in zip(rows, ctx):
        own_from = max(shared, _seen_from(c, r, n) // page)
        sink_pages = -(-min(c.get("sinks", 0), n) // page) if "window" in c else 0
        kept.append(sorted(set(range(min(sink_pages, -(-n // page)))) | set(range(own_from, -(-n // page)))))
    pages = shared + sum(len(k) for k in kept) + 2
    # Pages of a pool that other requests have used: any order.
    order = torch.randperm(pages, device=DEV, generator=gen).to(torch.int32)
    table = torch.full((c["b"], width), -1, dtype=torch.int32, device=DEV)
    table[:, :shared] = order[:shared]
    at = shared
    for b, own_pages in enumerate(kept):
        table[b, torch.tensor(own_pages, device=DEV)] = order[at:at + len(own_pages)]
        at += len(own_pages)
    s = dict(c=c, table=table, pages=pages, rows=rows, ctx=ctx, max_rows=max(rows), t=t)
    s["row_off"] = torch.tensor([sum(rows[:i]) for i in range(len(rows) + 1)], dtype=torch.int32, device=DEV)
    s["start"] = torch.tensor([n - r for n, r in zip(ctx, rows)], dtype=torch.int32, device=DEV)
    s["q"] = _rows(gen, t, c["hq"], d)
    if c["kind"] in ("write", "layer"):
        s["k"], s["v"] = _rows(gen, t, hkv, d), _rows(gen, t, hkv, d)
        s["wq"], s["wk"] = _weight(gen, d), _weight(gen, d)
        s["pos"] = torch.cat([_axis_positions(n - r, r, 3) for r, n in zip(rows, ctx)], dim=1)
        s["pos"] = s["pos"][0].contiguous() if c["axes"] == 1 else s["pos"]
    # What the pages hold: rows of unit size, keys as they are after rotation.
    s["old"] = [torch.randn((pages, hkv, page, d), device=DEV, generator=gen).to(torch.bfloat16) for _ in range(2)]
    return s


def prepare(case, seed):
    c = dict(case)
    s = _positions_inputs(c, seed) if c["kind"] == "positions" else _paged_inputs(c, seed)
    old = s.pop("old", None)
    if own:
        if c["kind"] in ("positions", "write", "layer"):
            from mtplx_amd.rotary import head_norms

            s["rotary"] = _table(c)
            s["norms"] = head_norms(s["wq"], s["wk"], eps=EPS) if c["norms"] else None
        if old is not None:
            from mtplx_amd.paged_kv_cache import PagedKVCache

            cache = PagedKVCache(s["pages"], c["hkv"], c["d"], page_size=c["page"], bits=c["bits"], device=DEV)
            every = torch.arange(s["pages"], dtype=torch.int32, device=DEV).unsqueeze(1)
            cache.write(*(x.transpose(1, 2).reshape(-1, c["hkv"], c["d"]) for x in old), every,
                        torch.zeros(s["pages"], dtype=torch.int32, device=DEV))
            s["cache"] = cache
        return s
    if c["kind"] in ("positions", "write", "layer"):
        s["freq"], s["axis"] = _frequencies(c.get("dims", c["d"])).to(DEV), _axis_of(c)
    if old is not None:
        s["pool"] = [_quantised(x) for x in old] if c["bits"] == 8 else old
    return s


# -- the plain form -------------------------------------------------------------

def _plain_heads(s, x, weight):
    """Rows [T, H, D]: each head normalised and rotated, in float32, rounded once."""
    c = s["c"]
    dims, trad = c.get("dims", c["d"]), c.get("trad", False)
    y = x.float()
    if c["norms"]:
        y = y * torch.rsqrt((y * y).mean(-1, keepdim=True) + EPS) * weight.float()
    pos = s["pos"].view(-1, x.shape[0])
    angle = pos[s["axis"]].t().double() * s["freq"]
    cs, sn = angle.cos().float().unsqueeze(1), angle.sin().float().unsqueeze(1)
    r = y[..., :dims]
    x1, x2 = (r[..., 0::2], r[..., 1::2]) if trad else (r[..., :dims // 2], r[..., dims // 2:])
    y1, y2 = x1 * cs - x2 * sn, x1 * sn + x2 * cs
    r = torch.stack([y1, y2], dim=-1).flatten(-2) if trad else torch.cat([y1, y2], dim=-1)
    return torch.cat([r, y[..., dims:]], dim=-1).to(x.dtype)


def _token_places(s):
    """(request, index in it, position) of each new token."""
    at = torch.arange(s["t"], device=DEV)
    b = torch.searchsorted(s["row_off"][1:].long(), at, right=True)
    i = at - s["row_off"].long()[b]
    return b, i, s["start"].long()[b] + i


def _plain_write(s):
    """The new rows into the pages; returns the finished queries."""
    c = s["c"]
    b, _, pos = _token_places(s)
    q, k = _plain_heads(s, s["q"], s["wq"]), _plain_heads(s, s["k"], s["wk"])
    page, slot = s["table"].long()[b, pos // c["page"]], pos % c["page"]
    for pool, x in zip(s["pool"], (k, s["v"])):
        if c["bits"] == 8:
            for part, value in zip(pool, _quantised(x)):
                part[page, :, slot] = value
        else:
            pool[page, :, slot] = x
    return q


def _plain_at(s, pool, pos):
    """float32 [B, Hkv, n, D] that the pages hold at positions [B, n] (no page: page 0's, masked later)."""
    c = s["c"]
    b = torch.arange(pos.shape[0], device=DEV).unsqueeze(1)
    page = s["table"].long()[b, (pos // c["page"]).clamp(max=s["table"].shape[1] - 1)].clamp(min=0)
    slot = pos % c["page"]
    if c["bits"] == 8:
        x = pool[0][page, :, slot].float() * pool[1][page, :, slot].unsqueeze(-1)
    else:
        x = pool[page, :, slot].float()
    return x.transpose(1, 2)


def _plain_read(s, start, count, lengths):
    """bf16 [B, Hkv, count, D] of the positions from start on, zeros from lengths on."""
    pos = start.long().unsqueeze(1) + torch.arange(count, device=DEV)
    live = pos < lengths.long().unsqueeze(1)
    pos = torch.where(live, pos, torch.zeros_like(pos))
    return tuple((_plain_at(s, pool, pos) * live[:, None, :, None]).to(torch.bfloat16).contiguous()
                 for pool in s["pool"])


def _padded_queries(s, q):
    """float32 [B, Hkv, rep, rows, D] of scaled queries, requests padded to the longest, and each row's position."""
    c = s["c"]
    top, rep = s["max_rows"], c["hq"] // c["hkv"]
    at = (s["row_off"][:-1].long().unsqueeze(1) + torch.arange(top, device=DEV)).clamp(max=s["t"] - 1)
    qp = q.float()[at].view(c["b"], top, c["hkv"], rep, c["d"]).permute(0, 2, 3, 1, 4)
    return qp * (1.0 / math.sqrt(c["d"])), s["start"].long().unsqueeze(1) + torch.arange(top, device=DEV)


def _packed_rows(s, o):
    """bf16 [T, Hq, D] of padded rows [B, Hkv, rep, rows, D]."""
    c = s["c"]
    b, i, _ = _token_places(s)
    return o.permute(0, 3, 1, 2, 4).reshape(c["b"], s["max_rows"], c["hq"], c["d"])[b, i].to(torch.bfloat16)


def _softmax_(score):
    """The weights in the scores' place, and their sum."""
    score -= score.amax(-1, keepdim=True)
    score = score.exp_()
    return score, score.sum(-1, keepdim=True)


def _plain_window(s, q):
    """The sinks' keys and those from the first token's window on, scored and masked."""
    c = s["c"]
    hkv, d, window, sinks = c["hkv"], c["d"], c["window"], c["sinks"]
    top = max(s["ctx"])
    first = (s["start"].long() - window + 1).clamp(min=min(sinks, top)).unsqueeze(1)
    pos = torch.cat([torch.arange(min(sinks, top), device=DEV).expand(c["b"], -1),
                     first + torch.arange(min(top, window - 1 + s["max_rows"]), device=DEV)], dim=1)
    k, v = (_plain_at(s, pool, pos) for pool in s["pool"])
    qp, at = _padded_queries(s, q)
    rep, rows = qp.shape[2:4]
    score = torch.matmul(qp.reshape(c["b"], hkv, rep * rows, d), k.transpose(2, 3).contiguous())
    score = score.view(c["b"], hkv, rep, rows, -1)
    j, p = pos.unsqueeze(1), at.unsqueeze(2)
    hidden = (j > p) | ((j <= p - window) & (j >= sinks))
    weight, total = _softmax_(score.masked_fill_(hidden[:, None, None], float("-inf")))
    o = torch.matmul(weight.view(c["b"], hkv, rep * rows, -1), v.contiguous()).view(c["b"], hkv, rep, rows, d)
    return _packed_rows(s, o / total)


def _plain_prefix(s, q):
    """The prefix's keys once for the rows of all requests, each tail for its own."""
    c = s["c"]
    b, hkv, d, shared = c["b"], c["hkv"], c["d"], c["prefix"] // c["page"] * c["page"]
    qp, at = _padded_queries(s, q)
    rep, rows = qp.shape[2:4]
    qp = qp.reshape(b, hkv, rep * rows, d)
    together = torch.arange(shared, device=DEV).unsqueeze(0)
    tail = shared + torch.arange(max(s["ctx"]) - shared, device=DEV)
    kp, vp = (_plain_at(s, pool, together)[0] for pool in s["pool"])
    kt, vt = (_plain_at(s, pool, tail.expand(b, -1)) for pool in s["pool"])
    every = qp.transpose(0, 1).reshape(hkv, b * rep * rows, d)
    score = torch.cat([torch.matmul(every, kp.transpose(1, 2).contiguous()).view(hkv, b, rep, rows, shared).transpose(0, 1),
                       torch.matmul(qp, kt.transpose(2, 3).contiguous()).view(b, hkv, rep, rows, -1)
                       .masked_fill_((tail > at.unsqueeze(2))[:, None, None], float("-inf"))], dim=-1)
    weight, total = _softmax_(score)
    o = torch.matmul(weight[..., :shared].transpose(0, 1).reshape(hkv, b * rep * rows, shared), vp.contiguous())
    o = o.view(hkv, b, rep, rows, d).transpose(0, 1)
    o = o + torch.matmul(weight[..., shared:].reshape(b, hkv, rep * rows, -1), vt.contiguous()).view(b, hkv, rep, rows, d)
    return _packed_rows(s, o / total)


# -- one pass -------------------------------------------------------------------

def _write(s):
    if not own:
        return _plain_write(s)
    return s["cache"].write(s["k"], s["v"], s["table"], s["start"], s["row_off"], max_rows=s["max_rows"],
                            queries=s["q"], rotary=s["rotary"], norms=s["norms"], positions=s["pos"])


def _window(s, q):
    c = s["c"]
    if not own:
        return _plain_window(s, q)
    from mtplx_amd.paged_attention import paged_sdpa

    return paged_sdpa(q, s["cache"], s["table"], s["start"], s["row_off"], max_rows=s["max_rows"], window=c["window"],
                      sinks=c["sinks"])


def run(state):
    s = state
    c = s["c"]
    if c["kind"] == "positions":
        if own:
            from mtplx_amd.rotary import apply_rotary

            return apply_rotary(s["rotary"], s["q"], s["k"], s["pos"], norms=s["norms"])
        return _plain_heads(s, s["q"], s["wq"]), _plain_heads(s, s["k"], s["wk"])
    if c["kind"] == "window":
        return _window(s, s["q"])
    if c["kind"] == "layer":
        return _window(s, _write(s))
    if c["kind"] == "prefix":
        if not own:
            return _plain_prefix(s, s["q"])
        from mtplx_amd.paged_attention import paged_sdpa

        return paged_sdpa(s["q"], s["cache"], s["table"], s["start"], s["row_off"], max_rows=s["max_rows"],
                          shared=c["prefix"] // c["page"] * c["page"])
    q = _write(s)
    ends = s["start"] + (s["row_off"][1:] - s["row_off"][:-1])
    if own:
        return q, s["cache"].read(s["table"], s["max_rows"], start=s["start"], lengths=ends)
    return q, _plain_read(s, s["start"], s["max_rows"], ends)


# -- from the definition, in 64 bits --------------------------------------------

def _exact_heads(c, x, weight, pos):
    """float64 rows [T, H, D] of a call's queries or keys at positions [axes, T]."""
    dims, trad = c.get("dims", c["d"]), c.get("trad", False)
    x = x.double()
    if c["norms"]:
        size = torch.linalg.vector_norm(x, dim=-1, keepdim=True)
        x = weight.double() * x / torch.sqrt(size * size / c["d"] + EPS)
    sections, turn = _sections(c)
    pairs = dims // 2
    if sections is None:
        axis = [0] * pairs
    elif turn:
        axis = [i % len(sections) if i // len(sections) < sections[i % len(sections)] else 0 for i in range(pairs)]
    else:
        axis = [a for a, n in enumerate(sections) for _ in range(n)]
    turned = torch.stack([pos[axis[i]].double() * 1.0e6 ** (-2.0 * i / dims) for i in range(pairs)], dim=1)
    z = torch.polar(torch.ones_like(turned), turned).unsqueeze(1)
    one, two = (slice(0, dims, 2), slice(1, dims, 2)) if trad else (slice(0, pairs), slice(pairs, dims))
    w = torch.complex(x[..., one], x[..., two]) * z
    y = x.clone()
    y[..., one], y[..., two] = w.real, w.imag
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
    if c["kind"] == "positions":
        s = _positions_inputs(c, seed)
        pos = s["pos"].view(c["axes"], -1)
        return _exact_heads(c, s["q"], s["wq"], pos), _exact_heads(c, s["k"], s["wk"], pos)
    s = _paged_inputs(c, seed)
    d, rep, page, bits = c["d"], c["hq"] // c["hkv"], c["page"], c["bits"]
    q, new = s["q"].double(), None
    if c["kind"] in ("write", "layer"):
        pos = s["pos"].view(c["axes"], -1)
        q = _exact_heads(c, s["q"], s["wq"], pos)
        new = [_exact_stored(x, bits) for x in (_exact_heads(c, s["k"], s["wk"], pos), s["v"].double())]
    if c["kind"] == "write":
        got = [torch.zeros((c["b"], c["hkv"], s["max_rows"], d), dtype=torch.float64, device=DEV) for _ in range(2)]
        for b, rows in enumerate(s["rows"]):
            lo = int(s["row_off"][b])
            for x, stored in zip(got, new):
                x[b, :, :rows] = stored[lo:lo + rows].transpose(0, 1)
        return q, tuple(got)
    if new is not None:
        q = q.to(torch.bfloat16).double()   # what a layer hands from the rotation to the attention
    out = []
    for b, (rows, ctx) in enumerate(zip(s["rows"], s["ctx"])):
        lo = int(s["row_off"][b])
        # Request b's own positions, those that no row sees among them (page 0's there).
        ids = s["table"][b, :-(-ctx // page)].long().clamp(min=0)
        kv = [_exact_stored(x[ids].transpose(0, 1).reshape(c["hkv"], -1, d)[:, :ctx].double(), bits) for x in s["old"]]
        if new is not None:
            for x, stored in zip(kv, new):
                x[:, ctx - rows:] = stored[lo:lo + rows].transpose(0, 1)
        o = torch.empty((rows, c["hq"], d), dtype=torch.float64, device=DEV)
        j, p = torch.arange(ctx, device=DEV), torch.arange(ctx - rows, ctx, device=DEV).unsqueeze(1)
        seen = j <= p
        if "window" in c:
            seen &= (j > p - c["window"]) | (j < c["sinks"])
        for h in range(c["hq"]):
            score = (q[lo:lo + rows, h] @ kv[0][h // rep].T) / math.sqrt(d)
            o[:, h] = torch.softmax(score.masked_fill(~seen, float("-inf")), dim=-1) @ kv[1][h // rep]
        out.append(o)
    return torch.cat(out)


def work(case):
    c = dict(case)
    if c["kind"] == "positions":
        n = c["t"] * (c["hq"] + c["hkv"]) * c["d"]
        return {"bytes": 4.0 * n + 4.0 * c["axes"] * c["t"], "flops": 3.0 * n * c["dims"] / c["d"] + 4.0 * n * c["norms"]}
    rows, ctx = _shape(c)
    t = sum(rows)
    row = c["hkv"] * (2 * c["d"] if c["bits"] == 16 else c["d"] + 4)   # one stored token of K or V
    made = 4.0 * t * (c["hq"] + c["hkv"]) * c["d"]                     # q in and out, k and v in
    if c["kind"] == "write":
        return {"bytes": made + 4.0 * t * row + 4.0 * t * c["hkv"] * c["d"],
                "flops": (3.0 + 4.0 * c["norms"]) * t * (c["hq"] + c["hkv"]) * c["d"]}
    keys, pairs = 0.0, 0.0
    for r, n in zip(rows, ctx):
        if c["kind"] == "prefix":
            keys += n - c["prefix"]
            pairs += r * (n - r) + r * (r + 1) / 2.0
            continue
        sinks, window = c["sinks"], c["window"]
        lo = max(0, n - r - window + 1)
        keys += n if sinks >= lo else sinks + n - lo
        # A token at p sees the last `window` positions and the sinks before them.
        pairs += sum(p + 1 if p < window else window + min(sinks, p + 1 - window) for p in range(n - r, n))
    keys += c.get("prefix", 0)
    moved = 2.0 * keys * row + 4.0 * t * c["hq"] * c["d"]
    if c["kind"] == "layer":
        moved += made
    return {"bytes": moved, "flops": 4.0 * pairs * c["hq"] * c["d"]}
