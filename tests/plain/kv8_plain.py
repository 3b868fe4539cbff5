"""The 8-bit cache and its block tables restated with Python integers and 64-bit floats, one block at a time."""
import math

import torch


def need(n, block, ring=0):
    return -(-(min(n, ring) if ring else n) // block)


def extend(slots, lengths, new, tables, held, free, count, block, ring, tokens):
    """Lists in, lists out: (status, cu_q, kv_len, positions, tok_seq, cache_rows, tables, held, count)."""
    rows = len(slots)
    tables, held = [list(t) for t in tables], list(held)
    bad = lambda code: (code, [0] * (rows + 1), [0] * rows, [-1] * tokens, [0] * tokens, [-1] * tokens, tables, held, count)
    live = [s for s in slots if s != -1]
    if any(n < 0 for n in new) or any(not 0 <= s < len(tables) for s in live) or len(set(live)) != len(live) or \
            any(s >= 0 and L < 0 for s, L in zip(slots, lengths)):
        return bad(4)
    if sum(new) > tokens:
        return bad(3)
    wants = [need(L + n, block, ring) if s >= 0 else 0 for s, L, n in zip(slots, lengths, new)]
    if any(w > len(tables[0]) for w in wants):
        return bad(2)
    if sum(max(0, w - held[s]) for s, w in zip(slots, wants) if s >= 0) > count:
        return bad(1)
    cu, kv_len, positions, seqs, out = [0], [], [], [], []
    for i, (s, L, n) in enumerate(zip(slots, lengths, new)):
        cu.append(cu[-1] + n)
        seqs += [i] * n
        if s < 0:
            kv_len.append(0)
            positions += [-1] * n
            out += [-1] * n
            continue
        kv_len.append(L + n)
        while held[s] < wants[i]:
            count -= 1
            tables[s][held[s]] = free[count]
            held[s] += 1
        for p in range(L, L + n):
            place = p % ring if ring else p
            kept = not ring or p // block + ring // block > (L + n - 1) // block
            positions.append(p)
            out.append(tables[s][place // block] * block + place % block if kept else -1)
    pad = tokens - cu[-1]
    return 0, cu, kv_len, positions + [-1] * pad, seqs + [0] * pad, out + [-1] * pad, tables, held, count


def scale_of(amax):
    """The least power of two, 2^-126 at least, with amax <= 127 of it; NaN where amax is not finite."""
    if not math.isfinite(amax):
        return math.nan
    e = -126
    while amax > 127.0 * 2.0 ** e:
        e += 1
    return 2.0 ** e


def write(x, rows, pages, scales):
    """x [tokens, heads, D] (any float type) to cache rows (-1: not kept), in order; ``pages`` float64 [blocks, heads, P, D]
    of whole numbers and ``scales`` float64, changed in place.  Tokens that follow each other in one block go in together."""
    P = pages.shape[2]
    x = x.double()
    t = 0
    while t < len(rows):
        if rows[t] < 0:
            t += 1
            continue
        b, p = divmod(rows[t], P)
        n = 1
        while t + n < len(rows) and p + n < P and rows[t + n] == rows[t] + n:
            n += 1
        for h in range(pages.shape[1]):
            piece = x[t:t + n, h]
            s = scale_of(float(piece.abs().max()) if bool(torch.isfinite(piece).all()) else math.inf)
            old = float(scales[b, h])
            if p and (math.isnan(old) or math.isnan(s)):
                s = math.nan
            elif p and old >= s:
                s = old
            elif p:
                pages[b, h, :p] = torch.round(pages[b, h, :p] * (old / s))        # (rounds halves to even)
            scales[b, h] = s
            pages[b, h, p:p + n] = 0.0 if math.isnan(s) else torch.round(piece / s)
        t += n


def first_kept(n, block, ring):
    return max(0, ((n - 1) // block - ring // block + 1) * block) if ring and n else 0


def read(pages, scales, table, positions, ring=0):
    """Values [positions, heads, D] of one sequence."""
    P = pages.shape[2]
    out = []
    for p in positions:
        place = p % ring if ring else p
        b = int(table[place // P])
        out.append(pages[b, :, place % P].double() * scales[b].double()[:, None])
    return torch.stack(out) if out else torch.zeros((0, pages.shape[1], pages.shape[3]), dtype=torch.float64)


def attend(q, keys, values, first, position, scale, cap, window):
    """One token: q [H, D] against keys/values [n, G, D] of positions first .. first + n - 1.  Returns [H, D]."""
    H, G = q.shape[0], keys.shape[1]
    out = torch.zeros((H, values.shape[2]), dtype=torch.float64)
    lo = max(first, position - window + 1 if window else 0)
    if lo > position:
        return out
    k, v = keys[lo - first:position + 1 - first], values[lo - first:position + 1 - first]
    for h in range(H):
        g = h // (H // G)
        if bool(torch.isnan(k[:, g]).any()) or bool(torch.isnan(v[:, g]).any()):
            out[h] = math.nan
            continue
        z = k[:, g] @ q[h].double() * scale
        if cap > 0:
            z = cap * torch.tanh(z / cap)
        out[h] = torch.softmax(z, 0) @ v[:, g]
    return out
