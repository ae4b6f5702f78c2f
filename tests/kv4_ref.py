"""Plain 64-bit forms of the operators on the 4-bit cache, element by element from the layout that
include/seedless_hip.h states (numpy, CPU)."""
import numpy as np


def places(page, dim):
    """Byte of each (token, dim) code and word of each (token, group) within a head's part of a page: key, key s|b, value, value s|b."""
    off, d = np.arange(page)[:, None], np.arange(dim)[None, :]
    codes, sbs = page * dim // 2, page * dim // 16
    key = off * (dim // 2) + (d % 64 // 16) * (dim // 8) + (d // 64) * 8 + d % 16 // 2
    part = dim // 16
    value = codes + sbs + ((off // 8 * 16 + d // part) * 8 + off % 8) * (dim // 32) + d % part // 2
    word = off * (dim // 64) + np.arange(dim // 64)[None, :]
    return key, codes // 4 + word, value, (2 * codes + sbs) // 4 + word


def unpack(pages, page, kv, dim):
    """uint8 [n_pages, bytes] -> dict of codes [n_pages * page, kv, dim], scale and bias [.., kv, dim / 64] (float64), for k and v."""
    n = pages.shape[0]
    heads = np.ascontiguousarray(pages).reshape(n, kv, -1)
    words = heads.view(np.uint32)
    key, ksb, value, vsb = places(page, dim)
    out = {}
    for name, at, sb in (("k", key, ksb), ("v", value, vsb)):
        code = (heads[:, :, at] >> (np.arange(dim) % 2 * 4).astype(np.uint8)) & 15
        w = words[:, :, sb]
        scale, bias = ((x & 0xffff).astype(np.uint16).view(np.float16).astype(np.float64) for x in (w, w >> 16))
        tok = lambda x: np.moveaxis(x, 1, 2).reshape(n * page, kv, -1)  # noqa: E731
        out[name] = dict(codes=tok(code), scale=tok(scale), bias=tok(bias))
    return out


def values(part):
    c = part["codes"].astype(np.float64)
    g = c.reshape(*c.shape[:-1], -1, 64)
    with np.errstate(invalid="ignore"):
        return (g * part["scale"][..., None] + part["bias"][..., None]).reshape(c.shape)


def pack(part_k, part_v, page, kv, dim):
    """The inverse of unpack: bytes [n_pages, ..]."""
    n = part_k["codes"].shape[0] // page
    heads = np.zeros((n, kv, page * 9 * dim // 8), np.uint8)
    key, ksb, value, vsb = places(page, dim)
    for part, at, sb in ((part_k, key, ksb), (part_v, value, vsb)):
        head = lambda x: np.moveaxis(x.reshape(n, page, kv, -1), 1, 2)  # noqa: E731
        code = head(part["codes"]).astype(np.uint8)
        heads[:, :, at[:, 0::2]] = code[..., 0::2] | (code[..., 1::2] << 4)
        word = head(part["scale"]).astype(np.float16).view(np.uint16).astype(np.uint32) | (head(part["bias"]).astype(np.float16).view(np.uint16).astype(np.uint32) << 16)
        heads.view(np.uint32)[:, :, sb] = word
    return heads.reshape(n, -1)


def quantise(x):
    """x [.., dim] float64 -> codes, scale, bias by the stated rule."""
    g = x.reshape(*x.shape[:-1], -1, 64)
    bad = ~np.isfinite(g).all(-1)
    g = np.clip(np.where(bad[..., None], 0.0, g), -65504, 65504)
    mn, mx = g.min(-1), g.max(-1)
    low = np.abs(mn) > np.abs(mx)
    scale = np.maximum((mx - mn) * (1 / 15), 1e-7) * np.where(low, 1, -1)      # the range times the double next to 1/15
    edge = np.where(low, mn, mx)
    n = np.rint(edge / scale)
    scale = np.where(n != 0, edge / np.where(n != 0, n, 1), scale).astype(np.float32).astype(np.float16).astype(np.float64)
    bias = np.where(n != 0, edge, 0.0).astype(np.float32).astype(np.float16).astype(np.float64)
    codes = np.clip(np.rint((g - bias[..., None]) / scale[..., None]), 0, 15)
    codes[bad] = 0
    return dict(codes=codes.reshape(x.shape).astype(np.uint8), scale=np.where(bad, np.nan, scale), bias=np.where(bad, np.nan, bias))


def turn(x, weight, cos, sin, pos, eps):
    """Norm and rotation of rows [t, heads, dim] in float64."""
    x = x.astype(np.float64)
    if weight is not None:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * weight.astype(np.float64)
    if cos is None:
        return x
    c, s = cos[pos][:, None].astype(np.float64), sin[pos][:, None].astype(np.float64)
    h = c.shape[-1]
    a, b = x[..., :h], x[..., h:2 * h]
    return np.concatenate((a * c - b * s, b * c + a * s, x[..., 2 * h:]), -1)


def plan(ctx, new, table, held, free, free_count, page, max_tokens):
    """Request after request, with a Python list as the free list."""
    n, width = table.shape
    ctx, new, held = ([int(v) for v in x] for x in (ctx, new, held))
    stack = [int(v) for v in free[:min(max(int(free_count[0]), 0), len(free))]]
    start, rows = [], 0
    sane = []
    for r in range(n):
        start.append(rows)
        k = max(new[r], 0)
        fits = k <= max_tokens - rows
        sane.append(fits and ctx[r] >= 0 and new[r] >= 0 and 0 <= held[r] <= width and ctx[r] + new[r] <= width * page and ctx[r] <= held[r] * page)
        rows = min(max_tokens, rows + k)
    start.append(rows)
    want = [-(-(ctx[r] + new[r]) // page) if sane[r] else held[r] for r in range(n)]
    out = np.full((n, width), -1, np.int32)
    for r in range(n):
        if sane[r]:
            stack += [int(table[r, c]) for c in range(want[r], held[r])]
    after, kv_len, unserved, short = [], [], 0, False
    slot, pos = np.full(max_tokens, -1, np.int32), np.zeros(max_tokens, np.int32)
    for r in range(n):
        keep = min(max(held[r], 0), width)
        need = max(want[r] - held[r], 0) if sane[r] else 0
        if sane[r]:
            keep = min(keep, want[r])
        out[r, :keep] = table[r, :keep]
        ok = sane[r] and (need == 0 or (not short and need <= len(stack)))
        if sane[r] and not ok:
            short = True
        if ok:
            for c in range(need):
                out[r, held[r] + c] = stack.pop()
            keep += need
        unserved += not ok
        after.append(keep)
        kv_len.append(ctx[r] + new[r] if ok else 0)
        for i in range(start[r + 1] - start[r]):
            t, p = start[r] + i, ctx[r] + i
            pos[t] = np.int64(p).astype(np.int32)
            if ok:
                slot[t] = out[r, p // page] * page + p % page
    left = np.full(len(free), -1, np.int32)
    left[:len(stack)] = stack
    i32 = lambda v: np.array(v, np.int32)  # noqa: E731
    return out, i32(after), left, i32([len(stack)]), i32(start), i32(kv_len), slot, pos, i32([unserved])


def attention(q, parts, table, q_start, kv_len, page, n_pages, scale, gate=None, max_rows=1 << 30, eps_out=2.0 ** -11):
    """softmax(scale q k^T) v and, beside it, how far a result may be off: rounding of the result (eps_out, half a step);
    weights that meet the values as fp16 (half a step 2^-11, or 2^-25 below fp16's normal numbers) in two parts, s * (code - 8)
    and b + 8 s, the second itself rounded to fp16; scores in fp32 over s * sum(q code) + b * sum(q); exp and the
    normaliser 2^-20.  Rows that are left alone come back as NaN in both."""
    t, heads, dim = q.shape
    k, v = values(parts["k"]), values(parts["v"])
    kv = k.shape[1]
    out, tol = (np.full((t, heads, dim), np.nan) for _ in range(2))
    wide = lambda x: np.repeat(x, 64, -1)  # noqa: E731
    for r in range(len(kv_len)):
        rows = q_start[r + 1] - q_start[r]
        for i in range(min(rows, max_rows)):
            at = q_start[r] + i
            j = np.arange(max(0, min(kv_len[r], table.shape[1] * page) - rows + i + 1))
            ids = table[r, j // page]
            j, ids = j[(ids >= 0) & (ids < n_pages)], ids[(ids >= 0) & (ids < n_pages)]
            at_slot = ids * page + j % page
            for h in range(heads):
                g = h // (heads // kv)
                if len(j) == 0:
                    out[at, h], tol[at, h] = 0.0, 0.0
                    continue
                qq = q[at, h].astype(np.float64)
                s = scale * (k[at_slot, g] @ qq)
                w = np.exp(s - s.max())
                total = w.sum()
                w /= total
                o = w @ v[at_slot, g]
                ks, kb, vs, vb = (np.abs(wide(parts[x][y][at_slot, g])) for x, y in (("k", "scale"), ("k", "bias"), ("v", "scale"), ("v", "bias")))
                rest = np.abs(wide(parts["v"]["bias"][at_slot, g] + 8 * parts["v"]["scale"][at_slot, g]))
                delta = 2.0 ** -24 * (dim + 8) * abs(scale) * ((15 * ks + kb) @ np.abs(qq)).max()
                e = 2.0 ** -11 * (w @ (8 * vs + 2 * rest)) + 2.0 ** -22 * len(j) / total + (2 * delta + 2.0 ** -20) * (w @ (np.abs(v[at_slot, g]) + 8 * vs))
                if gate is not None:
                    y = 1 / (1 + np.exp(-gate[at, h].astype(np.float64)))
                    o, e = o * y, e * y
                out[at, h], tol[at, h] = o, e + eps_out * np.abs(o) + 2.0 ** -25
    return out, tol
