"""The 4-bit cache's format in numpy, element by element as speech_kv.h defines it, and float64 attention with the error
bounds that follow from the kernels' roundings."""
import math

import numpy as np
import torch

GROUP, LIMIT = 32, np.float32(16384.0)
NIBBLE = (0, 4, 1, 5, 2, 6, 3, 7)
QUAD = (0, 2, 1, 3)


def quantise(x):
    """(codes [..., D], scale, low [..., D / 32] float16) of float32 rows."""
    x = np.asarray(x, np.float32)
    x = np.where(np.isnan(x), np.float32(0), np.clip(x, -LIMIT, LIMIT)).astype(np.float32)
    g = x.reshape(*x.shape[:-1], -1, GROUP)
    low = g.min(-1).astype(np.float16)
    span = (g.max(-1) - low.astype(np.float32)) * (np.float32(1) / np.float32(15))
    scale = np.maximum(span, np.float32(0)).astype(np.float16)
    with np.errstate(divide="ignore"):
        inv = np.where(scale > 0, np.float32(1) / scale.astype(np.float32), np.float32(0)).astype(np.float32)
    code = np.rint((g - low.astype(np.float32)[..., None]) * inv[..., None])
    return np.clip(code, 0, 15).astype(np.uint8).reshape(x.shape), scale, low


def values(code, scale, low):
    """float64 values of codes [..., D]."""
    g = code.reshape(*code.shape[:-1], -1, GROUP).astype(np.float64)
    return (low.astype(np.float64)[..., None] + scale.astype(np.float64)[..., None] * g).reshape(code.shape)


def write_row(pool, is_v, slot, head, code, scale, low):
    """One (token, head) row into a uint8 pool [blocks, heads, tiles, 10 D]."""
    tiles, width = pool.shape[2:]
    d = width // 10
    tile, t = slot // 16, slot % 16
    row = pool[tile // tiles, head, tile % tiles]
    half = row[8 * d:].view(np.float16)
    if not is_v:
        for c in range(d // 8):
            word = 0
            for j in range(8):
                word |= int(code[8 * c + j]) << (4 * NIBBLE[j])
            row[t * d // 2 + 4 * c:t * d // 2 + 4 * c + 4] = np.frombuffer(np.uint32(word).tobytes(), np.uint8)
        for g in range(d // GROUP):
            half[(t * (d // GROUP) + g) * 2:(t * (d // GROUP) + g) * 2 + 2] = scale[g], low[g]
    else:
        quad, k = t // 4, t % 4
        for m in range(d // 2):
            row[quad * 2 * d + 4 * m + k] = int(code[2 * m]) | int(code[2 * m + 1]) << 4
        for g in range(d // GROUP):
            at = (quad * (d // GROUP) + g) * 8 + QUAD[k]
            half[at], half[at + 4] = scale[g], low[g]


def read_row(pool, is_v, slot, head):
    """(code [D], scale, low [D / 32]) of one (token, head) row."""
    tiles, width = pool.shape[2:]
    d = width // 10
    tile, t = slot // 16, slot % 16
    row = pool[tile // tiles, head, tile % tiles]
    half = row[8 * d:].view(np.float16)
    code = np.zeros(d, np.uint8)
    if not is_v:
        for c in range(d // 8):
            word = int(np.frombuffer(row[t * d // 2 + 4 * c:t * d // 2 + 4 * c + 4].tobytes(), np.uint32)[0])
            for j in range(8):
                code[8 * c + j] = word >> (4 * NIBBLE[j]) & 15
        at = [(t * (d // GROUP) + g) * 2 for g in range(d // GROUP)]
        return code, half[at], half[[a + 1 for a in at]]
    quad, k = t // 4, t % 4
    for m in range(d // 2):
        b = int(row[quad * 2 * d + 4 * m + k])
        code[2 * m], code[2 * m + 1] = b & 15, b >> 4
    at = [(quad * (d // GROUP) + g) * 8 + QUAD[k] for g in range(d // GROUP)]
    return code, half[at], half[[a + 4 for a in at]]


def rotate64(x, table, positions, interleaved):
    """float64 rotation of rows x [N, H, D], and the sum of the two products' magnitudes (for bounds)."""
    half = table.shape[1] // 2
    cos, sin = table[positions][:, None, :half].double(), table[positions][:, None, half:].double()
    x = x.double()
    y, mag = x.clone(), x.abs()
    lo, hi = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if interleaved else (slice(0, half), slice(half, 2 * half))
    a, b = x[..., lo], x[..., hi]
    y[..., lo], y[..., hi] = a * cos - b * sin, b * cos + a * sin
    mag[..., lo], mag[..., hi] = (a * cos).abs() + (b * sin).abs(), (b * cos).abs() + (a * sin).abs()
    return y, mag


def attention64(q, k, v, visible, scale):
    """One head in float64: q [Q, D], k, v [T, D], query i sees the first visible[i] keys. (out [Q, D], weights [Q, T],
    scores)."""
    seen = torch.arange(k.shape[0], device=q.device)[None, :] < visible[:, None]
    s = (q @ k.T) * scale
    s = torch.where(seen, s, torch.full_like(s, -math.inf))
    w = torch.softmax(s, -1)
    w = torch.where(seen.any(-1, keepdim=True), w, torch.zeros_like(w))
    vv = torch.where(seen.any(0)[:, None], v, torch.zeros_like(v))
    return w @ vv, w, s


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def reference(q, held, table, visible, bs, blocks, scale):
    """Attention over a 4-bit cache, (out, bound) float64 [Q, H, D] of one row: q [Q, H, D], visible [Q] keys, held: (values
    [slots, H, D], scale, low [slots, H, D / 32]) of K and of V in float64."""
    (k, ks, _), (v, vs, vl) = held
    n_q, heads, d = q.shape
    group = heads // k.shape[1]
    t = int(visible.max().clamp(min=0))
    out, bound = (torch.zeros(n_q, heads, d, dtype=torch.float64, device="cuda") for _ in range(2))
    if t == 0:
        return out, bound
    pos = torch.arange(t, device="cuda")
    blk = table[pos // bs].long()
    good = (blk >= 0) & (blk < blocks)
    slot = blk.clamp(0, blocks - 1) * bs + pos % bs
    half = half_step(q.dtype)
    wide = lambda x: x.repeat_interleave(32, -1)
    for h in range(heads):
        qq = q[:, h].double()
        kk, vv = k[slot, h // group], v[slot, h // group]
        kk, vv = kk[good], vv[good]
        seen = [int((pos[good] < n).sum()) for n in visible.tolist()]
        if vv.shape[0] == 0:
            continue
        o, w, s = attention64(qq, kk, vv, torch.tensor(seen, device="cuda"), scale)
        # Scores: fp32 sums. 16-bit queries also sum their products with the codes' bases (at most 1040 scales each), and
        # their elements below 2^-14 of the greatest round to 2^-25 of it.
        mag = qq.abs() @ kk.abs().T
        if q.dtype == torch.float32:
            ds = (d + 8) * 2.0 ** -24 * mag
            dv = 2.0 ** -23 * vv.abs()
        else:
            ds = 2.0 ** -22 * (qq.abs() @ (1040 * wide(ks[slot, h // group])[good]).T) + 2.0 ** -22 * mag + \
                2.0 ** -24 * qq.abs().amax(-1, keepdim=True) * kk.abs().sum(-1)
            # V: one fp16 rounding about the group's middle and one of the middle.
            mid = wide(vl[slot, h // group] + 8 * vs[slot, h // group])[good]
            dv = 2.0 ** -11 * ((vv - mid).abs() + mid.abs()) * 1.01 + 2.0 ** -24
        ds = torch.where(w > 0, ds * abs(scale) + 2.0 ** -21 * s.abs() + 2.0 ** -21, torch.zeros_like(s))
        grow = torch.expm1(2 * ds.amax(-1, keepdim=True))  # weights' relative error, their sum's included
        absw = w @ vv.abs()
        out[:, h] = o
        bound[:, h] = w @ dv + grow * (absw + o.abs()) + half * o.abs() + 2.0 ** -20 * absw + 2.0 ** -25
    return out, bound
