"""Plain references of the paged-cache operators: whole numbers by a simulation of
the definition, values in 64 bits on the CPU (torch tensors in, torch out)."""
import math

import torch


def plan(context, new, table, free, num_free, page, most):
    """zs_paged_plan, one token after the other.  Returns (table, slots,
    sequences, positions, seqlens, cu_new, counts) as lists of ints."""
    table = [list(r) for r in table]
    width = len(table[0])
    left = free[:max(0, min(num_free, len(free)))]
    total_free = len(left)
    slots, seqs, poss, seqlens, cu = [], [], [], [], [0]
    missing = 0
    for b, (c, n) in enumerate(zip(context, new)):
        c, n = max(c, 0), max(n, 0)
        n = min(n, most - len(slots))
        held = -(-c // page)
        mine = {}
        for lp in range(held, -(-(c + n) // page)):
            if lp < width and left:
                mine[lp] = table[b][lp] = left.pop()
            else:
                missing += 1
        have = held + len(mine)
        for t in range(c, c + n):
            lp = t // page
            block = mine.get(lp, -1) if lp >= held else table[b][lp] if lp < width else -1
            slots.append(block * page + t % page if block >= 0 else -1)
            seqs.append(b)
            poss.append(t)
        seqlens.append(min(c + n, have * page))
        cu.append(len(slots))
    asked = sum(max(n, 0) for n in new)
    rest = [-1] * (most - len(slots))
    counts = [asked, total_free - len(left), missing, len(left)]
    return table, slots + rest, seqs + rest, poss + rest, seqlens, cu, counts


def append(k, v, k_cache, v_cache, slots, bounds=None):
    """zs_paged_append on CPU copies of the caches, in place."""
    blocks, page = k_cache.shape[:2]
    for i, s in enumerate(slots.tolist()):
        if not 0 <= s < blocks * page:
            continue
        block, off = divmod(s, page)
        k_cache[block, off], v_cache[block, off] = k[i], v[i]
    if bounds is None:
        return
    touched = {}
    for i, s in enumerate(slots.tolist()):
        if 0 <= s < blocks * page:
            touched.setdefault(s // page, []).append(i)
    def value(x):  # (fmin and fmax pass over quiet NaNs only)
        return torch.where(x.isnan(), math.nan, x.float())

    for block, rows in touched.items():
        x = value(k[rows])
        low, high = x[0], x[0]
        for y in x[1:]:
            low, high = torch.fmin(low, y), torch.fmax(high, y)
        if not any(int(slots[i]) == block * page for i in rows):
            old = value(bounds[block])
            low, high = torch.fmin(low, old[:, 0]), torch.fmax(high, old[:, 1])
        bounds[block, :, 0], bounds[block, :, 1] = low.to(bounds.dtype), high.to(bounds.dtype)


def scores(q, bounds, table, length, page, heads_k, b):
    """(Hkv, n) scores of sequence b's pages in 64 bits."""
    n = min(-(-max(length, 0) // page), table.shape[1])
    group = q.shape[1] // heads_k
    out = torch.full((heads_k, n), -math.inf, dtype=torch.float64)
    for p in range(n):
        block = int(table[b, p])
        if not 0 <= block < bounds.shape[0]:
            continue
        for h in range(heads_k):
            x = q[b, h * group:(h + 1) * group].double()
            lo, hi = bounds[block, h].double()
            s = (x.clamp(min=0) * hi + x.clamp(max=0) * lo).sum(1)
            s = torch.where(s.isnan(), torch.full_like(s, math.inf), s)
            out[h, p] = s.max()
    return out


def select(q, bounds, table, lens, page, top_k, sink=1, local=1):
    heads_k = bounds.shape[1]
    pages = torch.full((q.shape[0], heads_k, top_k), -1, dtype=torch.int32)
    for b, length in enumerate(lens):
        s = scores(q, bounds, table, length, page, heads_k, b)
        n = s.shape[1]
        for h in range(heads_k):
            order = sorted(range(n), key=lambda p: (not (p < sink or p >= n - local), -s[h, p], p))
            take = sorted(order[:top_k])
            pages[b, h, :len(take)] = torch.tensor(take, dtype=torch.int32)
    return pages


def attend(q, k_cache, v_cache, table, pages, lens, scale=None):
    """(out, lse, allowed error of out, allowed error of lse), all float64.

    The errors allowed: the output's rounding to bf16 (2^-8 of it); scores in fp32
    (a sum of D exact products, each addition off by 2^-24 of the sum of their
    sizes at most, and the scaling: (D + 4) 2^-24 of sum |q k| scale), which move a
    weight by twice that relatively at most, the normaliser included; weights
    that enter the product with 16 bits (2^-16); sums of T weights and of T
    products in fp32 with their rescalings and a merge of the splits, and the
    exponentials (3 T 2^-24 in all, T counted from 64)."""
    B, H, D = q.shape
    blocks, page, heads_k, _ = k_cache.shape
    group = H // heads_k
    scale = 1 / math.sqrt(D) if scale is None else scale
    out = torch.zeros(B, H, D, dtype=torch.float64)
    tol = torch.zeros(B, H, D, dtype=torch.float64)
    lse = torch.full((B, H), -math.inf, dtype=torch.float64)
    lse_tol = torch.zeros(B, H, dtype=torch.float64)
    for b in range(B):
        for h in range(heads_k):
            rows = []
            for lp in pages[b, h].tolist():
                if not 0 <= lp < table.shape[1] or not 0 <= int(table[b, lp]) < blocks:
                    continue
                live = min(max(int(lens[b]) - lp * page, 0), page)
                rows += [int(table[b, lp]) * page + i for i in range(live)]
            if not rows:
                continue
            k = k_cache.view(-1, heads_k, D)[rows, h].double()
            v = v_cache.view(-1, heads_k, D)[rows, h].double()
            x = q[b, h * group:(h + 1) * group].double()
            s = x @ k.t() * scale
            w = torch.softmax(s, 1)
            o = w @ v
            ds = (x.abs() @ k.abs().t()).amax(1, keepdim=True) * abs(scale) * (D + 4) * 2.0 ** -24
            many = 3 * max(len(rows), 64) * 2.0 ** -24
            at = slice(h * group, (h + 1) * group)
            out[b, at], lse[b, at] = o, torch.logsumexp(s, 1)
            tol[b, at] = 2.0 ** -8 * o.abs() + (w @ v.abs()) * (2 * ds + 2.0 ** -16 + many) + 1e-30
            lse_tol[b, at] = ds[:, 0] + many + 2.0 ** -22 * lse[b, at].abs()
    return out, lse, tol, lse_tol
