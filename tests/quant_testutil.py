"""Plain references of rotary positions and of the quantised paged cache, in 64 bits
on the CPU (torch tensors in, torch out)."""
import math

import numpy as np
import torch

EPS = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}    # half a step, relative
TINY = {torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25, torch.float32: 2.0 ** -150}  # and below the normal range


def rotary(x, positions, frequencies, factor=1.0, interleaved=False):
    """(x turned, allowed error) of (tokens, heads, dim), float64.

    The errors allowed: half a step of the type for the output; in fp32, cosine and sine
    (2^-24 each), one product's rounding and the sum's: 3 * 2^-24 of the two
    products' sizes; sine and cosine before their rounding 2^-33; the angle
    in 64 bits, three roundings of it here or there (2^-51 of the angle in all)."""
    pairs = len(frequencies)
    y = x.double()
    angle = positions.double()[:, None] * frequencies
    cos, sin = (angle.cos() * factor)[:, None], (angle.sin() * factor)[:, None]
    a, b = (y[..., 0:2 * pairs:2], y[..., 1:2 * pairs:2]) if interleaved else (y[..., :pairs], y[..., pairs:2 * pairs])
    u, v = a * cos - b * sin, b * cos + a * sin
    off = (2.0 ** -33 + 2.0 ** -51 * angle.abs())[:, None] * abs(factor) * (a.abs() + b.abs())
    du = 3 * 2.0 ** -24 * ((a * cos).abs() + (b * sin).abs()) + off
    dv = 3 * 2.0 ** -24 * ((b * cos).abs() + (a * sin).abs()) + off
    out, tol = y.clone(), torch.zeros_like(y)
    live = positions >= 0
    for at, z, d in ((0, u, du), (1, v, dv)):
        where = slice(at, 2 * pairs, 2) if interleaved else slice(at * pairs, (at + 1) * pairs)
        half = EPS[x.dtype] * (z.abs() + d) + TINY[x.dtype]
        out[..., where] = torch.where(live[:, None, None], z, y[..., where])
        tol[..., where] = torch.where(live[:, None, None], d + half, 0.0)
    return out, tol


def bf16_bits(x):
    return x.contiguous().view(torch.int16).numpy().view(np.uint16)


def quantize(x, bits):
    """Codes (n, D), scale and low as bf16 bits (n), of rows x (n, D) bf16."""
    most = 2 ** bits - 1
    codes, scales, lows = [], [], []
    for row in x.float().numpy():
        with np.errstate(all="ignore"):
            low = row.min()
            span = np.float32(row.max() - low)
        if not np.isfinite(row).all() or not np.isfinite(span):
            codes.append([0] * len(row))
            scales.append(0x7FC0)
            lows.append(0x7FC0)
            continue
        s = max((int((span / np.float32(most)).view(np.uint32)) >> 16) - 2, 0)
        value = lambda b: float(np.uint32(b << 16).view(np.float32))  # noqa: E731
        while most * value(s) < float(span):  # (exact in 64 bits)
            s += 1
        t = (row - low).astype(np.float32).astype(np.float64)
        codes.append(np.rint(t / value(s)).astype(int).tolist() if s else [0] * len(row))
        scales.append(s)
        lows.append(int(low.view(np.uint32)) >> 16)
    return np.array(codes, dtype=np.int64), np.array(scales), np.array(lows)


def places(dim, bits):
    """(byte, shift) of each channel's code in a row."""
    if bits == 8:
        return [(c, 0) for c in range(dim)]
    return [(c // 8 * 4 + bit // 8, bit % 8) for c in range(dim) for bit in [c % 2 * 16 + c % 8 // 2 * 4]]


def record_bytes(page, dim, bits):
    return page * (8 + dim * bits // 4)


def append(k, v, data, slots, page, dim, bits):
    """zs_paged_append_quant on a CPU copy of the pool (uint8 numpy), in place."""
    blocks, heads_k = data.shape[:2]
    row = dim * bits // 8
    for i, s in enumerate(slots.tolist()):
        if not 0 <= s < blocks * page:
            continue
        block, off = divmod(s, page)
        for side, x in enumerate((k, v)):
            codes, scale, low = quantize(x[i], bits)
            for h in range(heads_k):
                record = data[block, h]
                record[8 * off + 4 * side:][:4] = np.array([scale[h], low[h]], dtype=np.uint16).view(np.uint8)
                at = 8 * page + side * page * row + off * row
                record[at:at + row] = 0
                for c, (byte, shift) in enumerate(places(dim, bits)):
                    record[at + byte] |= int(codes[h, c]) << shift


def parts(data, page, dim, bits):
    """Codes, scales and lows of all rows: for key and value (codes (blocks, Hkv,
    page, D), scale, low (blocks, Hkv, page)), float64."""
    blocks, heads_k = data.shape[:2]
    row = dim * bits // 8
    byte, shift = np.array(places(dim, bits)).T
    side = data[..., :8 * page].reshape(blocks, heads_k, page, 8).copy().view(np.uint16).astype(np.uint32)
    out = []
    for i in range(2):
        codes = data[..., 8 * page + i * page * row:][..., :page * row].reshape(blocks, heads_k, page, row)
        c = codes[..., byte] >> shift & (2 ** bits - 1)
        s, m = ((side[..., 2 * i + j] << 16).view(np.float32).astype(np.float64) for j in range(2))
        out.append(tuple(torch.from_numpy(a) for a in (c.astype(np.float64), s, m)))
    return out


def read(data, slots, page, dim, bits):
    """zs_paged_read_quant: (k, v) bf16."""
    blocks, heads_k = data.shape[:2]
    out = torch.zeros(2, len(slots), heads_k, dim, dtype=torch.bfloat16)
    for side, (c, s, m) in enumerate(parts(data, page, dim, bits)):
        values = (c * s[..., None] + m[..., None]).float().to(torch.bfloat16)
        for i, slot in enumerate(slots.tolist()):
            if 0 <= slot < blocks * page:
                out[side, i] = values[slot // page, :, slot % page]
    return out[0], out[1]


def attend(q, data, table, lens, page, bits, scale=None):
    """(out (B, new, H, D), lse (B, H, new), allowed error of out, of lse), float64.

    The errors allowed: the output's rounding to bf16 (2^-8 of it); a score is s_k
    (q.c) + low_k sum(q) in fp32, with 16 + c in place of c in 4 bits and 16
    sum(q) taken off, D + 8 operations each off by 2^-24 of the sum of the sizes
    |q| (s_k (32 + c) + |low_k|) at most, which move a weight by twice that relatively at
    most, the normaliser included; sums of T weights and of T products of s_v (32 + c) +
    |low_v| in fp32 with their rescalings, the weights' scaling, a merge of the splits and
    the exponentials (3 T 2^-24 in all, T counted from 64).  A weight times s_v enters its
    product as two fp16: off by 2^-22 of it, which these cover, or by 2^-25 where the
    largest of them, s_v counting as 2^-30 at least, is 2^11 or more: T 2^bits 2^-36 2^-30
    besides what these cover."""
    B, new, H, D = q.shape
    blocks, heads_k = data.shape[:2]
    group = H // heads_k
    scale = 1 / math.sqrt(D) if scale is None else scale
    (kc, ks, km), (vc, vs, vm) = parts(data, page, D, bits)
    extra = 32.0 if bits == 4 else 0.0
    out = torch.zeros(B, new, H, D, dtype=torch.float64)
    tol = torch.zeros(B, new, H, D, dtype=torch.float64)
    lse = torch.full((B, H, new), -math.inf, dtype=torch.float64)
    lse_tol = torch.zeros(B, H, new, dtype=torch.float64)
    for b in range(B):
        for i in range(new):
            at = torch.arange(max(0, min(int(lens[b]) - new + 1 + i, table.shape[1] * page)))
            block = table[b].long()[at // page]
            seen = (block >= 0) & (block < blocks)
            block, off = block[seen], at[seen] % page
            if not len(block):
                continue
            for h in range(heads_k):
                rows = slice(h * group, (h + 1) * group)
                def take(c, s, m):
                    c, s, m = c[block, h, off], s[block, h, off][:, None], m[block, h, off][:, None]
                    return c * s + m, (c + extra) * s.abs() + m.abs()
                k, k_size = take(kc, ks, km)
                v, v_size = take(vc, vs, vm)
                x = q[b, i, rows].double()
                s = x @ k.t() * scale
                w = torch.softmax(s, 1)
                o = w @ v
                ds = (x.abs() @ k_size.t()).amax(1, keepdim=True) * abs(scale) * (D + 8) * 2.0 ** -24
                many = 3 * max(len(block), 64) * 2.0 ** -24
                out[b, i, rows], lse[b, rows, i] = o, torch.logsumexp(s, 1)
                tol[b, i, rows] = 2.0 ** -8 * o.abs() + (w @ v_size) * (2 * ds + many) + len(block) * 2.0 ** (bits - 66)
                lse_tol[b, rows, i] = ds[:, 0] + many + 2.0 ** -22 * lse[b, rows, i].abs()
    return out, lse, tol, lse_tol


def random_pool(g, blocks, heads_k, page, dim, bits, spread=1.0):
    """A pool of random codes; scales log-normal, lows so that values are spread around 0 (uint8 numpy)."""
    data = torch.randint(0, 256, (blocks, heads_k, record_bytes(page, dim, bits)), generator=g, dtype=torch.int32)
    data = data.to(torch.uint8).numpy()
    s = torch.randn(blocks, heads_k, page, 2, generator=g).mul(0.5 * spread).exp() * (3.0 / 2 ** bits)
    m = -s * 2 ** (bits - 1) * (1 + 0.2 * torch.randn(s.shape, generator=g))
    side = torch.stack([s, m], -1).to(torch.bfloat16)
    data[..., :8 * page] = bf16_bits(side).view(np.uint8).reshape(blocks, heads_k, 8 * page)
    return data
