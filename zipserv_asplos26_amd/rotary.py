"""Rotary positions: what turns the queries and keys of a step before they are
appended and attended to.

    frequencies, factor = rotary_frequencies(head_dim, base=500000.0, scaling="bands", stretch=8.0, trained=8192)
    q, k = apply_rotary(q, k, plan.positions, frequencies, factor=factor)

Pair i of a head's rotated channels turns by position * frequencies[i]; the
angles are made in 64 bits, so positions of millions lose nothing and no table of
positions is kept.
"""
from __future__ import annotations

import math

from ._lib import ZS_TYPE_BF16, ZS_TYPE_FP16, ZS_TYPE_FP32, check, lib
from .codec import _torch
from .paged import _check, _here, _MOST


def rotary_frequencies(rotated: int, base: float = 10000.0, scaling: str = "none", stretch: float = 1.0,
                       trained: int = 0, low_turns: float = 1.0, high_turns: float = 0.0, device="cuda"):
    """(frequencies, factor) of `apply_rotary` for the first `rotated` channels of a
    head (even): radians a position, float64 [rotated / 2], and what cosines and
    sines are multiplied by.

    w_i = base^(-2 i / rotated), and for contexts `stretch` times the `trained` positions, by
    `scaling`,
      "linear": all w_i / stretch (positions interpolated);
      "base":   base * stretch^(rotated / (rotated - 2)) for base, which divides the
                slowest pair by stretch and leaves the fastest;
      "bands":  a pair that turns high_turns times or more over the trained positions
                keeps w_i, one that turns low_turns times or less gets w_i / stretch,
                between them a share of each, linear in the turns (high_turns 0: 4);
      "ramp":   the same with a share linear in the pair's number, from the pair that
                turns high_turns times (0: 32), rounded down, to the one that turns
                low_turns times, rounded up, and the factor 0.1 ln(stretch) + 1."""
    torch = _torch()
    if rotated <= 0 or rotated % 2:
        raise ValueError(f"rotated must be a positive even number, got {rotated}")
    if not (base > 0 and stretch > 0):
        raise ValueError("base and stretch must be positive")
    if scaling not in ("none", "linear", "base", "bands", "ramp"):
        raise ValueError(f"scaling {scaling!r} is none of none, linear, base, bands, ramp")
    factor, pair = 1.0, torch.arange(rotated // 2, dtype=torch.float64)
    if scaling == "base":
        if rotated == 2:
            raise ValueError("a single pair has no base to scale")
        base = base * stretch ** (rotated / (rotated - 2))
    w = base ** (-2 * pair / rotated)
    if scaling == "linear":
        w = w / stretch
    elif scaling in ("bands", "ramp"):
        high = high_turns or (4.0 if scaling == "bands" else 32.0)
        if trained <= 0 or not 0 < low_turns < high:
            raise ValueError("trained must be positive and low_turns below high_turns")
        if scaling == "bands":
            keep = ((trained * w / (2 * math.pi) - low_turns) / (high - low_turns)).clamp(0, 1)
        else:
            if base == 1:
                raise ValueError("base must not be 1")

            def number(turns):  # of the pair that turns so often over the trained positions
                return rotated * math.log(trained / (2 * math.pi * turns)) / (2 * math.log(base))

            first = max(math.floor(number(high)), 0)
            last = min(math.ceil(number(low_turns)), rotated - 1)
            keep = 1 - ((pair - first) / max(last - first, 1e-3)).clamp(0, 1)
            factor = 0.1 * math.log(stretch) + 1.0 if stretch > 1 else 1.0
        w = w * keep + w / stretch * (1 - keep)
    return w.to(device), factor


def _apart(t):
    """Whether no two entries of t share a place."""
    reach = 0
    for step, size in sorted((s, n) for s, n in zip(t.stride(), t.shape) if n > 1):
        if step <= reach:
            return False
        reach += step * (size - 1)
    return True


def _meet(q, k, tokens, dim, size):
    """Whether tensors of `size` bytes an element that are turned in place, as `_side`
    gives them, may share one.  They do not where their addresses are apart, or, with the
    same stride, their rows of heads or, interleaved, their heads."""
    at, token, head, heads = q[0], q[1], q[2], q[6]
    k_at, k_token, k_head, k_heads = k[0], k[1], k[2], k[6]
    if not (tokens and heads and k_heads):
        return False
    off, row, k_row = (k_at - at) // size, (heads - 1) * head + dim, (k_heads - 1) * k_head + dim
    if off >= (tokens - 1) * token + row or -off >= (tokens - 1) * k_token + k_row:
        return False

    def apart(step, one, other):  # one each in every `step` elements
        return step > 0 and off % step >= one and off % step + other <= step

    if tokens > 1 and token != k_token:
        return True
    if tokens > 1 and apart(token, row, k_row):
        return False
    return not (head == k_head and apart(head, dim, dim) and (tokens == 1 or token % head == 0))


_ONE, _THREE, _FOUR = (None,), (None, None, None), (None, None, None, None)
_ABSENT = (0, 0, 0, 0, 0, 0, 0)


def _side(name, x, tokens, dim, inplace, torch):
    """The output of x, what is read for it, and both as the library takes them:
    address, token and head stride of each, heads."""
    shape, step = x.shape, x.stride()
    heads = shape[-2]
    rows = x
    if len(shape) == 4:
        if shape[0] > 1 and shape[1] > 1 and step[0] != shape[1] * step[1]:
            rows = None  # tokens that do not follow one stride
        else:
            step = step[1 if shape[1] > 1 else 0:][:1] + step[2:]
    if rows is None or (step[2] != 1 and dim > 1):
        if inplace:
            raise ValueError(f"{name} is turned in place: its tokens must follow one stride, its heads be contiguous")
        rows, step = x.contiguous(), (heads * dim, dim, 1)
    at = rows.data_ptr()
    if inplace:
        if not _apart(x):
            raise ValueError(f"{name} is turned in place: its heads must be apart")
        return x, rows, (at, step[0], step[1], at, step[0], step[1], heads)
    out = torch.empty(shape, dtype=x.dtype, device=x.device)
    return out, rows, (at, step[0], step[1], out.data_ptr(), heads * dim, dim, heads)


def apply_rotary(q, k, positions, frequencies, factor: float = 1.0, interleaved: bool = False,
                 inplace: bool = False):
    """q and k with their heads' first 2 * len(frequencies) channels turned by their
    tokens' positions: (q, k).  q: (tokens, H, D) or (B, new, H, D), k the same with its own
    heads, or None; bf16, fp16 or fp32, possibly slices of a fused projection's
    output.  positions: int32, one a token (`PagedPlan.positions`); a token with a
    negative one is copied as it is.  frequencies: float64 [pairs] on the GPU, radians
    a position; cosines and sines are multiplied by factor.

    Pair i is channels (i, i + pairs), with `interleaved` (2i, 2i + 1).  With `inplace` q
    and k are turned where they are (and returned), else into new contiguous tensors;
    in one buffer a token's heads of q then stand before or behind its heads of k, or the two
    alternate.  frequencies negated turn back what factor 1 has turned."""
    torch = _torch()
    if not isinstance(q, torch.Tensor):
        raise ValueError("q must be a bfloat16, float16 or float32 CUDA tensor")
    dtype = q.dtype
    type_ = ZS_TYPE_BF16 if dtype is torch.bfloat16 else ZS_TYPE_FP16 if dtype is torch.float16 else \
        ZS_TYPE_FP32 if dtype is torch.float32 else -1
    shape = q.shape
    four = len(shape) == 4
    if type_ < 0:
        raise ValueError("q must be a bfloat16, float16 or float32 CUDA tensor")
    _check(q, "q", dtype, _FOUR if four else _THREE, None, False)
    here = _here(q)
    if here is None:
        with torch.cuda.device(q.device):
            return apply_rotary(q, k, positions, frequencies, factor, interleaved, inplace)
    device, stream = here
    if four:
        lead, dim, tokens = (shape[0], shape[1]), shape[3], shape[0] * shape[1]
    else:
        lead, dim, tokens = (shape[0],), shape[2], shape[0]
    if k is not None:
        _check(k, "k", dtype, (*lead, None, dim), device, False)
    _check(positions, "positions", torch.int32, lead, device)
    _check(frequencies, "frequencies", torch.float64, _ONE, device)
    pairs = frequencies.shape[0]
    if pairs == 0 or 2 * pairs > dim:
        raise ValueError(f"{pairs} frequencies do not fit heads of {dim} channels")
    if tokens > _MOST:
        raise ValueError("there must be less than 2^31 tokens")
    q_out, q_in, q_args = _side("q", q, tokens, dim, inplace, torch)
    k_out, k_in, k_args = (None, None, _ABSENT) if k is None else _side("k", k, tokens, dim, inplace, torch)
    if inplace and k is not None and _meet(q_args, k_args, tokens, dim, q.element_size()):
        raise ValueError("q and k are turned in place: they must stand apart")
    # (q_in and k_in are held until the launch is queued)
    check("zs_rotary", lib().zs_rotary(stream, *q_args, *k_args, type_, positions.data_ptr(), tokens, dim,
                                       frequencies.data_ptr(), pairs, factor, bool(interleaved)))
    return q_out, k_out
