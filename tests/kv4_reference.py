"""Plain 64-bit forms of the prompt and 4-bit cache operators, and the cache's
layout read entry by entry, for their tests. Runs on any device."""
import math

import torch

BF = torch.bfloat16
BLOCK, GROUP = 16, 64


def quantise(x: torch.Tensor):
    """x [.., D] (fp32, taken as exact) -> codes (int64), s and m (bf16) per group of 64.
    s and m are rounded from fp32 as the definition says; codes in 64 bits, ties to even."""
    g = x.unflatten(-1, (-1, GROUP)).float()
    lo, hi = g.amin(-1, keepdim=True), g.amax(-1, keepdim=True)
    m = lo.to(BF)
    s = ((hi - lo) / torch.full_like(lo, 15.0)).to(BF)
    q = torch.where(s > 0, (g.double() - m.double()) / s.double().clamp_min(1e-300), torch.zeros_like(g).double())
    code = torch.nan_to_num(q, nan=0.0).round().clamp(0, 15)
    return code.flatten(-2).long(), s, m


def values(code, s, m):
    """The values codes stand for, in 64 bits."""
    return (code.unflatten(-1, (-1, GROUP)).double() * s.double() + m.double()).flatten(-2)


def rotate(x, cs):
    """x [T, heads, D] bf16, cs [T, D] bf16: the rotated pairs, rounded once to fp32."""
    h = x.shape[-1] // 2
    c, s = cs[:, None, :h].double(), cs[:, None, h:].double()
    a, b = x[..., :h].double(), x[..., h:].double()
    return torch.cat([a * c - b * s, b * c + a * s], -1).float()


def offsets(d, t, i):
    """Byte offset and nibble shift of the K and the V code, and byte offset of the K and the V pair, of token t, dimension i."""
    w = d // 32
    k = 4 * ((t * 4 + (i // 8) % 4) * w + i // 32) + (i % 8) // 2
    v = 9 * d + 4 * (((t // 8) * 32 + (i // 4) % 8 * 4 + (t % 8) // 2) * w + i // 32) + 2 * (t % 2) + (i % 4) // 2
    p = 4 * (t * (d // GROUP) + i // GROUP)
    return (k, (i % 2) * 4, 8 * d + p), (v, (i % 2) * 4, 17 * d + p)


def read_cache(cache, table, tokens, d):
    """K and V of the given tokens (1-D int64) of one slot: codes and values [tokens, hkv, D] each."""
    page = cache.shape[1] * BLOCK
    hkv = cache.shape[2]
    t = tokens[:, None, None]
    h = torch.arange(hkv, device=cache.device)[None, :, None]
    i = torch.arange(d, device=cache.device)[None, None, :]
    pg, tile = table.long()[t // page], t % page // BLOCK
    out = []
    for at, shift, pair in offsets(d, t % BLOCK, i):
        code = cache[pg, tile, h, at].long() >> shift & 15
        s, m = ((cache[pg, tile, h, pair + o].long() | cache[pg, tile, h, pair + o + 1].long() << 8).to(torch.int16).view(BF)
                for o in (0, 2))
        out.append((code, code.double() * s.double() + m.double()))
    return out


def write_cache(cache, table, tokens, k, v):
    """Quantises k and v [tokens, hkv, D] (fp32) into the slot's blocks (in place, on the cache's device)."""
    d = k.shape[-1]
    page = cache.shape[1] * BLOCK
    t = tokens[:, None, None]
    h = torch.arange(cache.shape[2], device=cache.device)[None, :, None]
    even = torch.arange(0, d, 2, device=cache.device)[None, None, :]
    grp = torch.arange(0, d, GROUP, device=cache.device)[None, None, :]
    pg, tile = table.long()[t // page], t % page // BLOCK
    for side, x in enumerate((k, v)):
        code, s, m = quantise(x)
        at = offsets(d, t % BLOCK, even)[side][0]
        cache[pg, tile, h, at] = (code[..., 0::2] | code[..., 1::2] << 4).to(torch.uint8)
        pair = offsets(d, t % BLOCK, grp)[side][2]
        for o, z in ((0, s), (2, m)):
            b = z.squeeze(-1).contiguous().view(torch.int16).long()
            cache[pg, tile, h, pair + o] = (b & 255).to(torch.uint8)
            cache[pg, tile, h, pair + o + 1] = (b >> 8 & 255).to(torch.uint8)


def attend(q, k, v, scale, visible=None):
    """One sequence in 64 bits: q [R, hq, D], k, v [L, hkv, D]; row r sees keys up to r + L - R
    (and only those of `visible` [L]). Keys a row does not see take no part, whatever they hold."""
    R, hq, d = q.shape
    L, hkv = k.shape[0], k.shape[1]
    out = torch.zeros(R, hq, d, dtype=torch.float64, device=q.device)
    for r in range(R):
        n = min(L, max(0, r + L - R + 1))
        keep = torch.arange(n, device=q.device) if visible is None else visible[:n].nonzero()[:, 0]
        if not keep.numel():
            continue
        for h in range(hq):
            s = (k[keep, h * hkv // hq].double() @ q[r, h].double()) * scale
            p = torch.softmax(s, 0)
            out[r, h] = p @ v[keep, h * hkv // hq].double()
    return out


def attend_fast(q, k, v, scale):
    """attend() without NaN or infinity in the inputs, all rows at once."""
    R, hq, d = q.shape
    L, hkv = k.shape[0], k.shape[1]
    if L == 0:
        return torch.zeros(R, hq, d, dtype=torch.float64, device=q.device)
    hidden = torch.arange(L, device=q.device)[None] > torch.arange(R, device=q.device)[:, None] + L - R
    out = torch.empty(R, hq, d, dtype=torch.float64, device=q.device)
    for h in range(hq):
        s = (q[:, h].double() @ k[:, h * hkv // hq].double().T) * scale
        p = torch.nan_to_num(torch.softmax(s.masked_fill(hidden, -math.inf), -1))
        out[:, h] = p @ v[:, h * hkv // hq].double()
    return out
