"""What is measured of the operators on a paged key/value cache that is held in 4 bits: plan (page tables and slots from
request lengths), append (norm and rotation of queries and keys, keys and values into the cache), attention over the
cache, read (cache rows as values).

A cache is a pool of pages; a page holds `page` tokens of every key/value head, and for each head, one behind the other,
  key codes [page][4][D/64][8 bytes]    token, quarter of a group of 64 dims, group: 16 dims, low nibble first
  key scale and bias [page][D/64] fp16 pairs
  value codes [page/8][16][8][D/32 bytes]    block of 8 tokens, sixteenth of the dims, token: D/16 dims, low nibble first
  value scale and bias [page][D/64] fp16 pairs
A value is scale * code + bias.  Slot page * `page` + offset names a token's place in the pool.

A case's lengths follow from its own numbers alone (`_lengths`), its values from the seed.
"""
import math
import random

import numpy as np
import torch

own = False

EPS = 1e-6
LOG = math.log
TYPES = {"float16": torch.float16, "bfloat16": torch.bfloat16}


# ---- cases ------------------------------------------------------------------------------------------------------------
def listed():
    lay = dict(heads=16, kv=2, dim=256, rot=64, dtype="float16")       # the engine's attention layers
    wide = dict(heads=32, kv=8, dim=128, rot=128, dtype="bfloat16")    # a generic grouped layout, rotated as a whole
    many = dict(heads=8, kv=8, dim=64, rot=32, dtype="bfloat16")       # every query head with its own keys
    return [
        # what a server does before every step of 32 lanes
        {"name": "plan_lanes32", "op": "plan", "requests": 32, "ctx_lo": 1024, "ctx_hi": 16384, "new_lo": 1, "new_hi": 1,
         "page": 64, "spare": 4096, "mix": 1},
        # a large server: prompts, single tokens, requests that ended (and give their pages back) in one step
        {"name": "plan_mixed1024", "op": "plan", "requests": 1024, "ctx_lo": 1, "ctx_hi": 32768, "new_lo": 0, "new_hi": 160,
         "page": 16, "spare": 65536, "mix": 2},
        # one new token of one sequence: latency alone
        {"name": "append_token", "op": "append", "requests": 1, "ctx_lo": 4095, "ctx_hi": 4095, "new_lo": 1, "new_hi": 1,
         "page": 64, "mix": 3, **lay},
        # a prompt chunk
        {"name": "append_chunk2048", "op": "append", "requests": 1, "ctx_lo": 4096, "ctx_hi": 4096, "new_lo": 2048, "new_hi": 2048,
         "page": 64, "mix": 4, **lay},
        # ragged prompts of several requests, many key/value heads
        {"name": "append_ragged_bf16", "op": "append", "requests": 9, "ctx_lo": 17, "ctx_hi": 8000, "new_lo": 331, "new_hi": 1500,
         "page": 16, "mix": 5, **wide},
        # batch-1 decode
        {"name": "decode_4k", "op": "attention", "requests": 1, "ctx_lo": 4095, "ctx_hi": 4095, "new_lo": 1, "new_hi": 1,
         "page": 64, "gate": True, "mix": 6, **lay},
        # 32 lanes at mixed contexts
        {"name": "decode_lanes32", "op": "attention", "requests": 32, "ctx_lo": 1024, "ctx_hi": 16384, "new_lo": 1, "new_hi": 1,
         "page": 64, "gate": True, "mix": 7, **lay},
        # rows of a speculative step, long contexts
        {"name": "verify_32k_bf16", "op": "attention", "requests": 6, "ctx_lo": 20001, "ctx_hi": 32768, "new_lo": 3, "new_hi": 5,
         "page": 16, "gate": False, "mix": 8, **wide},
        # a prompt from its first token
        {"name": "prefill_2048", "op": "attention", "requests": 1, "ctx_lo": 0, "ctx_hi": 0, "new_lo": 2048, "new_hi": 2048,
         "page": 64, "gate": True, "mix": 9, **lay},
        # chunks of several prompts behind what the cache already holds
        {"name": "chunks_bf16", "op": "attention", "requests": 3, "ctx_lo": 4001, "ctx_hi": 16000, "new_lo": 400, "new_hi": 1111,
         "page": 32, "gate": False, "mix": 10, **many},
        # a prompt prefix handed on as values
        {"name": "read_500", "op": "read", "requests": 1, "ctx_lo": 500, "ctx_hi": 500, "new_lo": 0, "new_hi": 0,
         "page": 64, "mix": 11, **lay},
        # four long sequences read out
        {"name": "read_long", "op": "read", "requests": 4, "ctx_lo": 3333, "ctx_hi": 16384, "new_lo": 0, "new_hi": 0,
         "page": 32, "mix": 12, **wide},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(LOG(lo), LOG(hi)))))))


def _ordered(rng, lo, hi):
    a, b = _log_int(rng, lo, hi), _log_int(rng, lo, hi)
    return min(a, b), max(a, b)


def draw(rng):
    op = rng.choice(["plan", "append", "append", "attention", "attention", "attention", "read"])
    page = rng.choice([16, 32, 64, 128])
    mix = rng.randrange(1 << 20)
    if op == "plan":
        lo, hi = _ordered(rng, 1, 32768)
        return {"op": op, "requests": _log_int(rng, 1, 900), "ctx_lo": lo, "ctx_hi": hi, "new_lo": 0, "new_hi": _log_int(rng, 1, 150),
                "page": page, "spare": _log_int(rng, 64, 60000), "mix": mix}
    kv, group, dim = rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 3, 4, 8]), rng.choice([64, 128, 256])
    lay = dict(heads=kv * group, kv=kv, dim=dim, rot=rng.choice([0, 16, 32, 64, dim]), dtype=rng.choice(["float16", "bfloat16"]))
    per = kv * dim
    if op == "append":
        n = _log_int(rng, 1, 8)
        hi = _log_int(rng, 1, max(1, 2048 * 512 // (per * n)))
        lo, top = _ordered(rng, 1, 16384)
        return {"op": op, "requests": n, "ctx_lo": lo, "ctx_hi": top, "new_lo": max(1, hi // 3), "new_hi": hi, "page": page, "mix": mix, **lay}
    if op == "read":
        n = _log_int(rng, 1, 8)
        lo, hi = _ordered(rng, 1, max(1, min(16384, 16384 * 1024 // (per * n))))
        return {"op": op, "requests": n, "ctx_lo": lo, "ctx_hi": hi, "new_lo": 0, "new_hi": 0, "page": page, "mix": mix, **lay}
    kind = rng.choice(["decode", "decode", "verify", "chunk"])
    gate = rng.random() < 0.5
    if kind == "chunk":
        n = _log_int(rng, 1, 3)
        new = _log_int(rng, 17, max(17, 2048 * 16 // (lay["heads"] * n)))
        lo, hi = _ordered(rng, 1, max(64, min(16000, (1 << 27) // (new * n * lay["heads"]))))
        return {"op": op, "requests": n, "ctx_lo": lo, "ctx_hi": hi, "new_lo": max(1, new // 3), "new_hi": new, "page": page, "gate": gate, "mix": mix, **lay}
    new = 1 if kind == "decode" else _log_int(rng, 2, 8)
    n = _log_int(rng, 1, 32)
    lo, hi = _ordered(rng, 1, max(16, min(32768, (1 << 27) // (per * n))))
    return {"op": op, "requests": n, "ctx_lo": lo, "ctx_hi": hi, "new_lo": min(new, 2 if new > 1 else 1), "new_hi": new, "page": page, "gate": gate, "mix": mix, **lay}


def _lengths(c):
    """(tokens already in the cache, new tokens) of each request: spread over the logarithm of the range, in mixed order."""
    r, n = random.Random(c["mix"]), c["requests"]
    out = []
    for lo, hi in ((c["ctx_lo"], c["ctx_hi"]), (c["new_lo"], c["new_hi"])):
        v = [int(round((lo + 1) * ((hi + 1) / (lo + 1)) ** ((i + 1) / n))) - 1 for i in range(n)]
        r.shuffle(v)
        out.append(v)
    if c["op"] == "plan" and n >= 64:                     # every 32nd request has ended
        out[0] = [0 if i % 32 == 5 else x for i, x in enumerate(out[0])]
        out[1] = [0 if i % 32 == 5 else x for i, x in enumerate(out[1])]
    return out


def _pages(tokens, page):
    return -(-tokens // page)


def work(c):
    ctx, new = _lengths(c)
    n, page = c["requests"], c["page"]
    if c["op"] == "plan":
        held = sum(_pages(x, page) for x in ctx)
        width = max(_pages(x + y, page) for x, y in zip(ctx, new)) + 4
        return {"bytes": 4 * (3 * n + held + c["spare"] + n * width + 3 * n + 2 * sum(new) + held + c["spare"]), "flops": 0}
    h, kv, d = c["heads"], c["kv"], c["dim"]
    cache = kv * (d + d // 8)                             # a token's keys and values with their scales and biases
    if c["op"] == "append":                               # with the new rows read back as values
        t = sum(new)
        return {"bytes": t * ((2 * h + 2 * kv) * d * 2 + 2 * cache + 2 * kv * d * 4), "flops": t * (h + 2 * kv) * d * 10}
    if c["op"] == "read":
        t = sum(ctx)
        return {"bytes": t * (cache + 2 * kv * d * 4), "flops": t * kv * d * 4}
    seen = sum(y * x + y * (y + 1) // 2 for x, y in zip(ctx, new))
    return {"bytes": (sum(ctx) + sum(new)) * cache + sum(new) * h * d * 2 * (3 if c["gate"] else 2), "flops": 4 * d * h * seen}


# ---- what a program has in hand --------------------------------------------------------------------------------------
def page_bytes(page, kv, dim):
    return page * kv * (dim + dim // 8)


def _fill(pool, page, kv, dim, gen):
    """Codes as quantised rows have them (bell-shaped over the sixteen steps) and scales of either sign."""
    view = _regions(pool, page, kv, dim)
    for key in ("k", "v"):
        codes = view[key]
        a = torch.empty(codes.shape, device="cuda", dtype=torch.float16)
        byte = None
        for shift in (0, 4):
            a.normal_(7.5, 3.2, generator=gen)
            nib = a.round().clamp_(0, 15).to(torch.uint8)
            byte = nib if byte is None else byte | (nib << shift)
        codes.copy_(byte)
        sb = view[key + "sb"].view(torch.float16).unflatten(-1, (dim // 64, 2))
        mag = torch.empty(sb.shape[:-1], device="cuda").uniform_(0.22, 0.42, generator=gen)
        side = torch.where(torch.rand(mag.shape, device="cuda", generator=gen) < 0.5, 1.0, -1.0)
        edge = torch.empty_like(mag).uniform_(6.4, 8.6, generator=gen)
        sb[..., 0] = (mag * side).half()
        sb[..., 1] = (-mag * side * edge).half()


def prepare(case, seed):
    c = case
    gen = torch.Generator(device="cuda").manual_seed(seed)
    cpu = torch.Generator().manual_seed(seed)
    ctx, new = _lengths(c)
    n, page = c["requests"], c["page"]
    i32 = dict(device="cuda", dtype=torch.int32)
    s = {"case": c, "page": page, "ctx": torch.tensor(ctx, **i32), "new": torch.tensor(new, **i32), "tokens": sum(new), "max_new": max(new)}
    if c["op"] == "plan":
        held = [_pages(x, page) for x in ctx]
        for i in range(5, n, 32):                          # ended requests still hold pages, others were cut back
            held[i] += 3
        for i in range(7, n, 16):
            held[i] += 1
        width = max(_pages(x + y, page) for x, y in zip(ctx, new)) + 4
        total = sum(held) + c["spare"]
        order = torch.randperm(total, generator=cpu).to(torch.int32)
        table = torch.full((n, width), -1, dtype=torch.int32)
        at = 0
        for i, k in enumerate(held):
            table[i, :k] = order[at:at + k]
            at += k
        free = torch.full((total,), -1, dtype=torch.int32)
        free[: c["spare"]] = order[at:]
        s |= {"table": table.cuda(), "held": torch.tensor(held, **i32), "free": free.cuda(), "free_count": torch.tensor([c["spare"]], **i32)}
        return s
    dim, kv, heads, dtype = c["dim"], c["kv"], c["heads"], TYPES[c["dtype"]]
    total = [x + y for x, y in zip(ctx, new)]
    count = [_pages(x, page) for x in total]
    width, pages = max(count), sum(count) + 3
    order = torch.randperm(pages, generator=cpu).to(torch.int32)
    table = torch.full((n, width), -1, dtype=torch.int32)
    at = 0
    for i, k in enumerate(count):
        table[i, :k] = order[at:at + k]
        at += k
    pool = torch.zeros(pages, page_bytes(page, kv, dim), device="cuda", dtype=torch.uint8)
    s |= {"pool": pool, "heads": heads, "kv": kv, "dim": dim, "table": table.cuda(), "kv_len": torch.tensor(total, **i32),
          "q_start": torch.tensor([0] + list(np.cumsum(new)), **i32), "max_kv": max(total)}
    rows = new if c["op"] != "read" else ctx               # appended rows, or all that are read
    first = ctx if c["op"] != "read" else [0] * n
    pos = torch.cat([torch.arange(a, a + k) for a, k in zip(first, rows)])
    req = torch.repeat_interleave(torch.arange(n), torch.tensor(rows))
    s["pos"] = pos.to(torch.int32).cuda()
    s["slot"] = (table[req, pos // page].long() * page + pos % page).to(torch.int32).cuda()
    if c["op"] != "append":
        _fill(pool, page, kv, dim, gen)
    if c["op"] == "attention":
        s["q"] = (torch.randn(s["tokens"], heads, dim, device="cuda", generator=gen) * 1.2).to(dtype)
        both = torch.randn(s["tokens"], heads, 2 * dim, device="cuda", generator=gen).to(dtype)    # a projection's [query | gate] per head
        s["gate"] = both[:, :, dim:] if c["gate"] else None
        s["scale"] = dim ** -0.5
    if c["op"] == "append":
        rot = c["rot"]
        # a projection's row: queries, keys, values side by side
        qkv = torch.randn(s["tokens"], (heads + 2 * kv) * dim, device="cuda", generator=gen) * 1.5
        qkv[:, ::37] *= 6.0                                # channels that stand out, as keys have them
        qkv = qkv.to(dtype)
        s["q"] = qkv[:, : heads * dim].unflatten(1, (heads, dim))
        s["k"] = qkv[:, heads * dim:(heads + kv) * dim].unflatten(1, (kv, dim))
        s["v"] = qkv[:, (heads + kv) * dim:].unflatten(1, (kv, dim))
        s["q_weight"] = (1 + 0.1 * torch.randn(dim, device="cuda", generator=gen)).to(dtype)
        s["k_weight"] = (1 + 0.1 * torch.randn(dim, device="cuda", generator=gen)).to(dtype)
        s["cos"] = s["sin"] = None
        if rot:
            angle = torch.arange(max(total), device="cuda", dtype=torch.float64)[:, None] * torch.exp(
                -torch.arange(rot // 2, device="cuda", dtype=torch.float64) * (2.0 / rot * LOG(1e7)))
            s["cos"], s["sin"] = angle.cos().float(), angle.sin().float()
    return s


# ---- plain forms -----------------------------------------------------------------------------------------------------
def _regions(pool, page, kv, dim):
    """Views of a pool's four parts, by page and head."""
    heads = pool.unflatten(1, (kv, -1))
    codes, sb = page * dim // 2, page * dim // 16
    k, ksb, v, vsb = heads.split([codes, sb, codes, sb], dim=2)
    return {"k": k.unflatten(2, (page, 4, dim // 64, 8)), "ksb": ksb.unflatten(2, (page, dim // 16)),
            "v": v.unflatten(2, (page // 8, 16, 8, dim // 32)), "vsb": vsb.unflatten(2, (page, dim // 16))}


def _nibbles(b):
    return torch.stack((b & 15, b >> 4), dim=-1).flatten(-2)


def _values(codes, sb, dim, dtype):
    """codes [..., dim] and bytes [..., dim / 16] of scale and bias -> scale * code + bias"""
    sb = sb.contiguous().view(torch.float16).unflatten(-1, (dim // 64, 2)).to(dtype)
    return (codes.unflatten(-1, (dim // 64, 64)).to(dtype) * sb[..., :1] + sb[..., 1:]).flatten(-2)


def _page_values(pool, ids, page, kv, dim, dtype):
    """Keys and values [..., page, kv, dim] of whole pages."""
    got = {}
    for key, part in _regions(pool, page, kv, dim).items():
        got[key] = part[ids]
    lead = ids.dim()
    k = _nibbles(got["k"]).transpose(-3, -2).flatten(-3)                     # [.., kv, page, dim]
    v = _nibbles(got["v"]).transpose(-3, -2).flatten(-2).flatten(-3, -2)     # [.., kv, page / 8, 8, 16, dim / 16]
    k, v = _values(k, got["ksb"], dim, dtype), _values(v, got["vsb"], dim, dtype)
    return k.transpose(lead, lead + 1), v.transpose(lead, lead + 1)


def _read_plain(s, dtype=torch.float32):
    page, kv, dim = s["page"], s["kv"], s["dim"]
    slot = s["slot"].long()
    at, off = slot // page, slot % page
    r = _regions(s["pool"], page, kv, dim)
    k = _nibbles(r["k"][at, :, off]).transpose(-3, -2).flatten(-3)
    v = _nibbles(r["v"][at, :, off // 8, :, off % 8]).flatten(-2)
    return _values(k, r["ksb"][at, :, off], dim, dtype), _values(v, r["vsb"][at, :, off], dim, dtype)


def _turn(x, weight, cos, sin, pos):
    x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * weight.to(x.dtype)
    if cos is None:
        return x
    c, sn = cos[pos][:, None].to(x.dtype), sin[pos][:, None].to(x.dtype)
    half = c.shape[-1]
    a, b, rest = x[..., :half], x[..., half:2 * half], x[..., 2 * half:]
    return torch.cat((a * c - b * sn, b * c + a * sn, rest), dim=-1)


def _quantise(x):
    """x [t, kv, dim] in 64 bits -> codes [t, kv, dim] and scales and biases [t, kv, dim / 64] as fp16"""
    g = x.clamp(-65504, 65504).unflatten(-1, (-1, 64))
    mn, mx = g.amin(-1, keepdim=True), g.amax(-1, keepdim=True)
    low = mn.abs() > mx.abs()
    scale = ((mx - mn) / 15).clamp_min(1e-7)
    scale = torch.where(low, scale, -scale)
    edge = torch.where(low, mn, mx)
    steps = (edge / scale).round()
    some = steps != 0
    scale = torch.where(some, edge / torch.where(some, steps, torch.ones_like(steps)), scale).float().half()
    bias = torch.where(some, edge, torch.zeros_like(edge)).float().half()
    codes = ((g - bias.double()) / scale.double()).round().clamp(0, 15).to(torch.uint8).flatten(-2)
    return codes, scale.squeeze(-1), bias.squeeze(-1)


def _append_plain(s):
    page, kv, dim = s["page"], s["kv"], s["dim"]
    pos, slot = s["pos"].long(), s["slot"].long()
    at, off = slot // page, slot % page
    q = _turn(s["q"].float(), s["q_weight"], s["cos"], s["sin"], pos).to(s["q"].dtype)
    k = _turn(s["k"].double(), s["k_weight"], s["cos"], s["sin"], pos)
    r = _regions(s["pool"], page, kv, dim)
    for key, x in (("k", k), ("v", s["v"].double())):
        codes, scale, bias = _quantise(x)
        pair = codes.unflatten(-1, (-1, 2))
        byte = pair[..., 0] | (pair[..., 1] << 4)
        if key == "k":
            r["k"][at, :, off] = byte.unflatten(-1, (dim // 64, 4, 8)).transpose(-3, -2)
        else:
            r["v"][at, :, off // 8, :, off % 8] = byte.unflatten(-1, (16, dim // 32))
        r[key + "sb"][at, :, off] = torch.stack((scale, bias), dim=-1).flatten(-2).view(torch.uint8)
    return (q, *_read_plain(s))


def _attention_plain(s):
    page, kv, dim, n = s["page"], s["kv"], s["dim"], s["ctx"].numel()
    heads, new, most = s["heads"], s["new"].long(), s["max_new"]
    k, v = _page_values(s["pool"], s["table"].long().clamp_min(0), page, kv, dim, torch.float32)
    k, v = (x.flatten(1, 2)[:, : s["max_kv"]] for x in (k, v))                       # [n, keys, kv, dim]
    row = torch.arange(most, device="cuda")
    at = (s["q_start"][:-1, None].long() + row).clamp_max(s["tokens"] - 1)
    q = s["q"].float()[at].unflatten(2, (kv, -1)).permute(0, 2, 1, 3, 4).flatten(2, 3).flatten(0, 1)   # [n * kv, most * group, dim]
    score = torch.bmm(q.contiguous(), k.permute(0, 2, 3, 1).flatten(0, 1).contiguous()) * s["scale"]
    seen = torch.arange(s["max_kv"], device="cuda") <= (s["kv_len"].long() - new)[:, None, None] + row[:, None]
    score = score.view(n, kv, most, heads // kv, -1).masked_fill_(~seen[:, None, :, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    p = (score - top).exp_()
    total = p.sum(-1, keepdim=True)
    v = torch.where((torch.arange(s["max_kv"], device="cuda") < s["kv_len"][:, None])[:, :, None, None], v, 0.0)
    o = torch.bmm(p.view(n * kv, most * (heads // kv), -1), v.transpose(1, 2).flatten(0, 1).contiguous())
    o = (o.view(n, kv, most, heads // kv, dim) / total).permute(0, 2, 1, 3, 4).flatten(2, 3)
    o = o[(row < new[:, None])]
    if s["gate"] is not None:
        o = o * (1 / (1 + (-s["gate"].float()).exp()))
    return o.to(s["q"].dtype)


def _plan_plain(s):
    page, table, free, n = s["page"], s["table"], s["free"].long(), s["ctx"].numel()
    ctx, new, held = s["ctx"].long(), s["new"].long(), s["held"].long()
    width, count = table.shape[1], free.numel()
    want = (ctx + new + page - 1) // page
    extra, need = (held - want).clamp_min(0), (want - held).clamp_min(0)
    have = s["free_count"].long() + extra.sum()
    upto = need.cumsum(0)
    fits = (need == 0) | (upto <= have)
    col = torch.arange(width, device="cuda")
    # the free pages, those given back behind them in the requests' order
    back = (col >= want[:, None]) & (col < held[:, None])
    index = torch.arange(count, device="cuda")
    given = (extra.cumsum(0) - extra)[:, None] + col - want[:, None] + s["free_count"].long()
    pool = free.clone()
    pool[given[back]] = table.long()[back]
    left = have - (need * fits).sum()
    # new pages come off the end
    grow = fits[:, None] & (col >= held[:, None]) & (col < want[:, None])
    taken = (have - 1 - (upto - need)[:, None] - (col - held[:, None])).clamp(0, count - 1)
    after = torch.where(fits, want, held)
    out = torch.where(grow, pool[taken], torch.where(col < torch.minimum(held, after)[:, None], table.long(), -1))
    pool = torch.where(index < left, pool, -1)
    start = torch.cat((torch.zeros(1, device="cuda", dtype=torch.long), new.cumsum(0)))
    token = torch.arange(s["tokens"], device="cuda")
    req = torch.searchsorted(start[1:], token, right=True)
    pos = ctx[req] + token - start[req]
    slot = torch.where(fits[req], out[req, (pos // page).clamp_max(width - 1)] * page + pos % page, -1)
    got = (out, after, pool, left, start, torch.where(fits, ctx + new, 0), slot, pos, (~fits).sum().view(1))
    return tuple(x.to(torch.int32) for x in got)


def run(s):
    op = s["case"]["op"]
    if own:
        from qwisp_amd import kv4
        if op == "plan":
            return tuple(kv4.plan(s["ctx"], s["new"], s["table"], s["held"], s["free"], s["free_count"], s["page"], s["tokens"]))
        cache = kv4.Pool(s["pool"], s["page"], s["kv"], s["dim"])
        if op == "append":
            q = kv4.append(cache, s["q"], s["k"], s["v"], s["slot"], s["pos"], s["cos"], s["sin"], s["q_weight"], s["k_weight"], eps=EPS)
            return (q, *kv4.read(cache, s["slot"]))
        if op == "read":
            return kv4.read(cache, s["slot"])
        return kv4.attention(cache, s["q"], s["table"], s["q_start"], s["kv_len"], max_rows=s["max_new"], max_keys=s["max_kv"],
                             scale=s["scale"], gate=s["gate"])
    return {"plan": _plan_plain, "append": _append_plain, "read": _read_plain, "attention": _attention_plain}[op](s)


# ---- the definition, in 64 bits ----------------------------------------------------------------------------------------
def _cache_rows(s, slots):
    """Keys and values [kv, rows, dim] in 64 bits, by where each dim's nibble lies."""
    page, kv, dim = s["page"], s["kv"], s["dim"]
    slots = slots.long()
    d = torch.arange(dim, device="cuda")
    off, at = (slots % page)[:, None], (slots // page)[:, None, None]
    head = torch.arange(kv, device="cuda")[:, None, None] * (page * (dim + dim // 8))
    group, quarter, in16 = d // 64, d % 64 // 16, d % 16
    part = dim // 16
    key = off * (dim // 2) + (quarter * (dim // 64) + group) * 8 + in16 // 2
    value = page * (dim // 2 + dim // 16) + ((off // 8 * 16 + d // part) * 8 + off % 8) * (part // 2) + d % part // 2
    rows = s["pool"][at.squeeze(-1).squeeze(-1)]                                        # [rows, bytes of a page]
    out = []
    for where, sb in ((key, page * dim // 2), (value, page * (dim + dim // 16))):
        place = (head + where).transpose(0, 1).flatten(1)                               # [rows, kv * dim]
        code = (rows.gather(1, place).view(-1, kv, dim) >> (d % 2 * 4).to(torch.uint8) & 15).double()
        base = (head.view(-1, 1) + sb + off[:, :, None] * (dim // 16) + group * 4)       # [rows, kv, dim]
        pick = lambda k: (rows.gather(1, (base + 2 * k).flatten(1)).int() | rows.gather(1, (base + 2 * k + 1).flatten(1)).int() << 8).to(torch.int16).view(torch.float16).double().view(-1, kv, dim)  # noqa: E731
        out.append((pick(0) * code + pick(1)).transpose(0, 1))
    return out


def exact(case, seed):
    if case["op"] == "plan":
        return None                                       # whole numbers: the plain form's own
    s = prepare(case, seed)
    page, kv, dim = s["page"], s["kv"], s["dim"]
    if case["op"] == "read":
        got = [[], []]
        for part in s["slot"].split(4096):
            for to, x in zip(got, _cache_rows(s, part)):
                to.append(x.transpose(0, 1))
        return tuple(torch.cat(x) for x in got)
    if case["op"] == "append":
        out = []
        for x, weight in ((s["q"], s["q_weight"]), (s["k"], s["k_weight"]), (s["v"], None)):
            y = x.double()
            if weight is not None:
                y = y / ((y ** 2).sum(-1, keepdim=True) / dim + EPS).sqrt() * weight.double()
                if s["cos"] is not None:
                    angle = torch.complex(s["cos"].double(), s["sin"].double())[s["pos"].long()][:, None]
                    half = angle.shape[-1]
                    z = torch.complex(y[..., :half].contiguous(), y[..., half:2 * half].contiguous()) * angle
                    y = torch.cat((z.real, z.imag, y[..., 2 * half:]), -1)
            if x is not s["q"]:                           # to the nearest of the sixteen values that a group can hold
                g = y.reshape(*y.shape[:-1], dim // 64, 64)
                small, large = g.min(-1).values, g.max(-1).values
                far = torch.where(small.abs() > large.abs(), small, large)
                step = torch.maximum((large - small) / 15, torch.full_like(far, 1e-7)) * torch.where(small.abs() > large.abs(), 1.0, -1.0)
                count = torch.round(far / step)
                step = torch.where(count == 0, step, far / count).float().half().double()
                first = torch.where(count == 0, 0.0, far).float().half().double()
                steps = torch.tensor([*range(0, 16, 2), *range(1, 16, 2)], device="cuda", dtype=torch.float64)  # halfway: the even one
                held = first[..., None, None] + step[..., None, None] * steps
                y = torch.empty_like(g)
                for i in range(0, g.shape[0], 256):
                    best = (g[i:i + 256, ..., None] - held[i:i + 256]).abs().argmin(-1)
                    y[i:i + 256] = held[i:i + 256].expand(*best.shape, 16).gather(-1, best[..., None]).squeeze(-1)
                y = y.flatten(-2)
            out.append(y)
        return tuple(out)
    group = s["heads"] // kv
    out = torch.empty(s["tokens"], s["heads"], dim, device="cuda", dtype=torch.float64)
    start, length, table = s["q_start"].tolist(), s["kv_len"].tolist(), s["table"].long()
    for r, keys in enumerate(length):
        rows = start[r + 1] - start[r]
        j = torch.arange(keys, device="cuda")
        slots = table[r, j // page] * page + j % page
        parts = [_cache_rows(s, x) for x in slots.split(4096)]
        k, v = (torch.cat([p[i] for p in parts], dim=1) for i in (0, 1))                 # [kv, keys, dim]
        for first in range(0, rows, 256):
            last = min(rows, first + 256)
            q = s["q"][start[r] + first:start[r] + last].double()
            hidden = j[None, :] > keys - rows + torch.arange(first, last, device="cuda")[:, None]
            for h in range(s["heads"]):
                w = (q[:, h] @ k[h // group].T * s["scale"]).masked_fill(hidden, -math.inf).softmax(-1)
                out[start[r] + first:start[r] + last, h] = w @ v[h // group]
    if s["gate"] is not None:
        out = out * torch.sigmoid(s["gate"].double())
    return out
