"""The operators for prompts and for a key/value cache held in 4 bits, as cases to measure.

    prompt   causal attention of packed sequences with grouped heads, each behind an optional prefix of keys
    append   rotary positions for q and k, and k and v appended to the paged 4-bit cache; the pages written
             come back as the values they stand for
    cached   attention of each slot's newest rows over its paged 4-bit cache

A cache block holds 16 tokens of one kv head in 18 * D bytes: codes of K (8 D), their (scale, minimum) pairs (D),
codes of V (8 D), their pairs (D). A group is 64 dimensions of one token: m = bf16(min), s = bf16((max - min) / 15),
code = round((x - m) / s) in 0..15, value = s * code + m.
"""
import math
import random

import torch

own = False

BF16 = torch.bfloat16
BLOCK = 16   # tokens of a cache block
GROUP = 64   # dimensions that share a scale and a minimum


# ---- cases -------------------------------------------------------------------------------------

def listed():
    return [
        # the newest token of a few requests over unpaged keys: the single-token form
        dict(name="prompt single tokens", op="prompt", n=4, q_lo=1, q_hi=1, pre_lo=15, pre_hi=600, hq=32, hkv=8, d=128, mix=1),
        # prefill chunks of at most 16 tokens behind what their slots hold (the mixed step)
        dict(name="prompt chunks", op="prompt", n=8, q_lo=1, q_hi=16, pre_lo=256, pre_hi=768, hq=32, hkv=8, d=128, mix=2),
        # whole prompts of different lengths, packed
        dict(name="prompt packed", op="prompt", n=16, q_lo=17, q_hi=2048, pre_lo=0, pre_hi=0, hq=32, hkv=8, d=128, mix=3),
        # as many key heads as query heads, 64 wide
        dict(name="prompt heads of 64", op="prompt", n=5, q_lo=129, q_hi=2000, pre_lo=0, pre_hi=0, hq=16, hkv=16, d=64, mix=4),
        # one long prompt
        dict(name="prompt long", op="prompt", n=1, q_lo=8191, q_hi=8191, pre_lo=0, pre_hi=0, hq=32, hkv=8, d=128, mix=5),
        # one decoded token of each of 28 slots
        dict(name="append single tokens", op="append", n=28, q_lo=1, q_hi=1, pre_lo=256, pre_hi=768, hq=32, hkv=8, d=128, page=16, mix=6),
        # chunks of long prompts behind what their slots hold, larger pages, heads of 64
        dict(name="append chunks", op="append", n=16, q_lo=16, q_hi=512, pre_lo=1, pre_hi=4096, hq=8, hkv=2, d=64, page=32, mix=7),
        # fresh prompts
        dict(name="append prompts", op="append", n=4, q_lo=500, q_hi=4000, pre_lo=0, pre_hi=0, hq=32, hkv=8, d=128, page=16, mix=8),
        # one slot, a short context
        dict(name="cached one slot", op="cached", n=1, q_lo=1, q_hi=1, pre_lo=65, pre_hi=65, hq=32, hkv=8, d=128, page=16, mix=9),
        # the decode step of 28 slots
        dict(name="cached decode", op="cached", n=28, q_lo=1, q_hi=1, pre_lo=256, pre_hi=768, hq=32, hkv=8, d=128, page=16, mix=10),
        # drafted tokens of 28 slots at long contexts
        dict(name="cached drafts", op="cached", n=28, q_lo=2, q_hi=5, pre_lo=1024, pre_hi=4096, hq=32, hkv=8, d=128, page=16, mix=11),
        # a few very long contexts
        dict(name="cached longest", op="cached", n=16, q_lo=1, q_hi=1, pre_lo=16384, pre_hi=32768, hq=32, hkv=8, d=128, page=64, mix=12),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    op = rng.choice(["prompt", "append", "cached"])
    d = rng.choice([64, 128, 128])
    hkv = rng.choice([1, 2, 4, 8])
    hq = hkv * rng.choice([1, 2, 3, 4, 5, 8])
    c = dict(op=op, hq=hq, hkv=hkv, d=d, mix=rng.randrange(1 << 20))
    if op == "prompt":
        c["n"] = _log(rng, 1, 32)
        top = int(math.sqrt(8191.0 ** 2 * 32 / (max(hq, 8) * c["n"])))  # the padded scores of the largest listed case
        c["q_hi"] = _log(rng, 1, min(top, 8191))
        c["q_lo"] = _log(rng, 1, c["q_hi"])
        c["pre_hi"] = rng.choice([0, _log(rng, 1, max(1, min(8191, top * top // c["q_hi"]) - c["q_hi"] + 1))])
        c["pre_lo"] = rng.randint(0, c["pre_hi"])
        return c
    c["page"] = rng.choice([16, 16, 32, 64])
    c["n"] = _log(rng, 1, 64)
    if op == "append":
        c["q_hi"] = _log(rng, 1, min(4000, 16000 // c["n"]))
        c["q_lo"] = _log(rng, 1, c["q_hi"])
        c["pre_hi"] = rng.choice([0, _log(rng, 1, 8000)])
        c["pre_lo"] = rng.randint(0, c["pre_hi"])
        return c
    c["q_hi"] = rng.choice([1, 1, rng.randint(1, 16)])
    c["q_lo"] = rng.randint(1, c["q_hi"])
    c["pre_hi"] = _log(rng, 1, min(32768, 16 * 32768 // (c["n"] * c["q_hi"])))
    c["pre_lo"] = rng.randint(0, c["pre_hi"])
    return c


def _lens(case):
    """New rows of each sequence, and the tokens ahead of them."""
    rng = random.Random(case["mix"])
    q = [rng.randint(case["q_lo"], case["q_hi"]) for _ in range(case["n"])]
    pre = [rng.randint(case["pre_lo"], case["pre_hi"]) for _ in range(case["n"])]
    return q, pre


def work(case):
    q, pre = _lens(case)
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    tq, tk = sum(q), sum(q) + sum(pre)
    seen = sum(a * b + a * (a + 1) // 2 for a, b in zip(q, pre))  # (row, key) pairs under the mask
    if case["op"] == "prompt":
        return {"bytes": 2 * d * (2 * tq * hq + 2 * tk * hkv), "flops": 4 * d * hq * seen}
    if case["op"] == "cached":
        return {"bytes": 4 * d * tq * hq + tk * hkv * 18 * d // BLOCK, "flops": 4 * d * hq * seen}
    page = case["page"]
    window = sum(a + b % page for a, b in zip(q, pre))  # tokens of the pages that are written
    held = window - tq
    fresh = case["pre_hi"] == 0
    moved = 2 * d * tq * (2 * hq + (3 if fresh else 2) * hkv) + tq * hkv * 18 * d // BLOCK + 2 * d * tq
    return {"bytes": moved + held * hkv * 18 * d // BLOCK + 4 * d * hkv * window, "flops": 3 * d * tq * (hq + hkv) + 8 * d * tq * hkv}


# ---- inputs ------------------------------------------------------------------------------------

def _pack(kc, kp, vc, vp):
    """Codes [.., 16, D] (uint8) and (scale, minimum) pairs [.., 16, D / 64, 2] (bf16) to blocks [.., 18 D]."""
    lead, d = kc.shape[:-2], kc.shape[-1]
    w = d // 32
    k = kc.reshape(-1, 16, w, 4, 8).permute(0, 1, 3, 2, 4).reshape(-1, 8 * d, 2)
    v = vc.reshape(-1, 2, 4, 2, w, 8, 4).permute(0, 1, 5, 2, 4, 3, 6).reshape(-1, 8 * d, 2)
    k, v = k[..., 0] | (k[..., 1] << 4), v[..., 0] | (v[..., 1] << 4)
    kp, vp = (p.contiguous().view(torch.uint8).reshape(-1, d) for p in (kp, vp))
    return torch.cat([k, kp, v, vp], -1).reshape(*lead, 18 * d)


def _unpack(blocks, d):
    """The inverse of _pack."""
    lead, w = blocks.shape[:-1], d // 32
    b = blocks.reshape(-1, 18 * d)

    def nibbles(x):
        return torch.stack([x & 15, x >> 4], -1)
    kc = nibbles(b[:, :8 * d]).reshape(-1, 16, 4, w, 8).permute(0, 1, 3, 2, 4).reshape(*lead, 16, d)
    vc = nibbles(b[:, 9 * d:17 * d]).reshape(-1, 2, 8, 4, w, 2, 4).permute(0, 1, 3, 5, 4, 2, 6).reshape(*lead, 16, d)
    kp, vp = (b[:, o:o + d].contiguous().view(BF16).reshape(*lead, 16, d // GROUP, 2) for o in (8 * d, 17 * d))
    return kc, kp, vc, vp


def _quantise(x):
    """x [.., D] in 32 bits to codes (uint8) and (scale, minimum) pairs in bf16."""
    g = x.unflatten(-1, (-1, GROUP))
    lo, hi = g.amin(-1, keepdim=True), g.amax(-1, keepdim=True)
    m, s = lo.to(BF16), ((hi - lo) / torch.full_like(lo, 15.0)).to(BF16)
    code = torch.where(s > 0, (g - m.float()) / s.float(), torch.zeros_like(g)).round().clamp(0, 15).to(torch.uint8)
    return code.flatten(-2), torch.cat([s, m], -1)


def _values(codes, pairs):
    """The values that codes and pairs stand for, in 32 bits."""
    g = codes.unflatten(-1, (-1, GROUP)).float()
    return (g * pairs[..., :1].float() + pairs[..., 1:].float()).flatten(-2)


def _cos_sin(max_pos, d, device):
    inv = 500000.0 ** (-torch.arange(0, d, 2, dtype=torch.float64, device=device) / d)
    a = torch.outer(torch.arange(max_pos, dtype=torch.float64, device=device), inv)
    return torch.cat([a.cos(), a.sin()], -1).to(BF16)


def _normal(g, *shape, dtype=BF16):
    return torch.randn(*shape, generator=g, device=g.device).to(dtype)


def prepare(case, seed):
    device = torch.device("cuda", torch.cuda.current_device())
    g = torch.Generator(device=device).manual_seed(seed)
    q, pre = _lens(case)
    n, hq, hkv, d = case["n"], case["hq"], case["hkv"], case["d"]
    tq = sum(q)
    st = dict(op=case["op"], q=q, pre=pre, n=n, hq=hq, hkv=hkv, d=d, scale=1.0 / math.sqrt(d))
    if case["op"] == "prompt":
        tk = tq + sum(pre)
        st["query"] = _normal(g, tq, hq, d)
        st["key"] = _normal(g, tk, hkv, d)
        if any(pre):
            st["value"] = _normal(g, tk, hkv, d)
        else:  # a fresh prompt's values lie in the rows of the fused projection
            st["value"] = _normal(g, tk, (hq + 2 * hkv) * d)[:, (hq + hkv) * d:].unflatten(-1, (hkv, d))
        st["k_lens"] = [a + b for a, b in zip(q, pre)]
        return st
    page = case["page"]
    longest = max(a + b for a, b in zip(q, pre))
    per = -(-longest // page)
    pages = n * per
    st |= dict(page=page, longest=longest)
    st["tables"] = torch.randperm(pages, generator=g, device=device).to(torch.int32).reshape(n, per)
    st["cache"] = torch.zeros(pages, page // BLOCK, hkv, 18 * d, dtype=torch.uint8, device=device)
    st["lens"] = torch.tensor(pre, dtype=torch.int32, device=device)
    # what the slots hold already (the newest rows too, where they are only read), made slot by slot
    bias = 2.0 * _normal(g, 2, hkv, 1, d, dtype=torch.float32)
    for i in range(n):
        held = pre[i] + (q[i] if case["op"] == "cached" else 0)
        tiles = -(-held // page) * (page // BLOCK)
        x = _normal(g, 2, tiles, hkv, BLOCK, d, dtype=torch.float32) + bias[:, None]
        (kc, kp), (vc, vp) = _quantise(x[0]), _quantise(x[1] * 0.5)
        st["cache"][st["tables"][i, :tiles * BLOCK // page].long()] = _pack(kc, kp, vc, vp).reshape(-1, page // BLOCK, hkv, 18 * d)
    if case["op"] == "cached":
        st["query"] = _normal(g, tq, hq * d)
        st["out"] = torch.empty(tq, hq * d, dtype=BF16, device=device)
        return st
    st["qkv"] = _normal(g, tq, (hq + 2 * hkv) * d)
    st["cos_sin"] = _cos_sin(longest + page, d, device)
    st["fresh"] = case["pre_hi"] == 0
    st["start"] = [b - b % page for b in pre]                       # each slot's window: the pages that are written
    st["count"] = [a + b % page for a, b in zip(q, pre)]
    st["q_rot"] = torch.empty(tq, hq * d, dtype=BF16, device=device)
    st["k_rot"] = torch.empty(tq, hkv * d, dtype=BF16, device=device)
    st["k_win"], st["v_win"] = (torch.empty(sum(st["count"]), hkv, d, dtype=BF16, device=device) for _ in range(2))
    return st


# ---- one pass ----------------------------------------------------------------------------------

def run(st):
    if st["op"] == "prompt":
        return _own_prompt(st) if own else _plain_prompt(st)
    if st["op"] == "append":
        return _own_append(st) if own else _plain_append(st)
    return _own_cached(st) if own else _plain_cached(st)


def _own_prompt(st):
    from swarmlora_b200 import worker_ops as wo
    return wo.prompt_attention(st["query"], st["key"], st["value"], st["q"], st["k_lens"], scale=st["scale"])


def _own_append(st):
    from swarmlora_b200 import worker_ops as wo
    k_rot = st["k_rot"] if st["fresh"] else None
    wo.kv4_append(st["qkv"], st["tables"], st["cache"], st["lens"], st["q_rot"], st["cos_sin"], st["hq"], st["hkv"],
                  head_dim=st["d"], page=st["page"], rows=st["q"], k_rot=k_rot)
    wo.kv4_gather(st["tables"], st["cache"], st["start"], st["count"], st["k_win"], st["v_win"], st["hkv"],
                  head_dim=st["d"], page=st["page"])
    return [st["q_rot"], st["k_win"], st["v_win"]] + ([k_rot] if st["fresh"] else [])


def _own_cached(st):
    from swarmlora_b200 import worker_ops as wo
    wo.paged_attention_kv4(st["q"], st["tables"], st["cache"], st["lens"], st["out"], st["query"], st["hq"], st["hkv"],
                           st["longest"], st["scale"], head_dim=st["d"], page=st["page"])
    return st["out"]


def _ragged(lens, device):
    """Of packed rows: each one's sequence, and its place in it."""
    t = torch.tensor(lens, device=device)
    seq = torch.repeat_interleave(torch.arange(len(lens), device=device), t, output_size=sum(lens))
    first = torch.cumsum(t, 0) - t
    return seq, torch.arange(sum(lens), device=device) - first[seq]


def _attend(q, k, v, q_lens, k_lens, scale):
    """q [n, hq, R, D], k and v [n, hkv, L, D] in 32 bits, padded; row r of sequence i sees keys up to r + k_len - q_len."""
    n, hq, r, d = q.shape
    hkv, ln = k.shape[1], k.shape[2]
    s = (q.reshape(n, hkv, -1, d) @ k.transpose(-1, -2)).reshape(n, hq, r, ln).mul_(scale)
    ql, kl = torch.tensor(q_lens, device=q.device), torch.tensor(k_lens, device=q.device)
    last = torch.arange(r, device=q.device) + (kl - ql)[:, None]
    hidden = torch.arange(ln, device=q.device) > last[..., None]
    s.masked_fill_(hidden[:, None], -math.inf)
    s.sub_(s.amax(-1, keepdim=True)).exp_()
    s.div_(s.sum(-1, keepdim=True))
    return (s.reshape(n, hkv, -1, ln) @ v).reshape(n, hq, r, d)


def _padded(x, seq, at, n, longest):
    out = torch.zeros(n, longest, *x.shape[1:], dtype=torch.float32, device=x.device)
    out[seq, at] = x.float()
    return out.transpose(1, 2).contiguous()


def _plain_prompt(st):
    n, device = st["n"], st["query"].device
    qs, qa = _ragged(st["q"], device)
    ks, ka = _ragged(st["k_lens"], device)
    q = _padded(st["query"], qs, qa, n, max(st["q"]))
    k = _padded(st["key"], ks, ka, n, max(st["k_lens"]))
    v = _padded(st["value"], ks, ka, n, max(st["k_lens"]))
    return _attend(q, k, v, st["q"], st["k_lens"], st["scale"])[qs, :, qa].to(BF16)


def _plain_cached(st):
    n, hq, hkv, d, device = st["n"], st["hq"], st["hkv"], st["d"], st["query"].device
    qs, qa = _ragged(st["q"], device)
    kc, kp, vc, vp = _unpack(st["cache"][st["tables"].long()], d)  # [n, pages, page / 16, hkv, 16, D]

    def held(codes, pairs):
        x = _values(codes, pairs).permute(0, 3, 1, 2, 4, 5).reshape(n, hkv, -1, d)[:, :, :st["longest"]]
        return x
    q = _padded(st["query"].reshape(-1, hq, d), qs, qa, n, max(st["q"]))
    o = _attend(q, held(kc, kp), held(vc, vp), st["q"], [a + b for a, b in zip(st["q"], st["pre"])], st["scale"])
    return o[qs, :, qa].reshape(-1, hq * d).to(BF16)


def _rotate(x, cs):
    """x [T, heads, D], cs [T, D]: pairs (i, i + D / 2) turned by their angles."""
    h = x.shape[-1] // 2
    c, s = cs[:, None, :h].float(), cs[:, None, h:].float()
    a, b = x[..., :h].float(), x[..., h:].float()
    return torch.cat([a * c - b * s, b * c + a * s], -1)


def _plain_append(st):
    hq, hkv, d, page, device = st["hq"], st["hkv"], st["d"], st["page"], st["qkv"].device
    pre = torch.tensor(st["pre"], device=device)
    seq, at = _ragged(st["q"], device)
    pos = at + pre[seq]
    x = st["qkv"].unflatten(-1, (-1, d))
    cs = st["cos_sin"][pos]
    q, k, v = _rotate(x[:, :hq], cs), _rotate(x[:, hq:hq + hkv], cs), x[:, hq + hkv:].float()
    (kc, kp), (vc, vp) = _quantise(k), _quantise(v)
    # the blocks of each slot's window, unpacked, changed and packed again
    tiles = [-(-c // BLOCK) for c in st["count"]]
    ts, ta = _ragged(tiles, device)
    first = torch.tensor(st["start"], device=device) // BLOCK
    tile = ta + first[ts]
    per = page // BLOCK
    where = (st["tables"].long()[ts, tile // per], tile % per)
    old = _unpack(st["cache"][where], d)  # [tiles, hkv, 16, ..]
    begin = torch.cumsum(torch.tensor(tiles, device=device), 0) - torch.tensor(tiles, device=device)
    row = begin[seq] + pos // BLOCK - first[seq]
    new = [o.transpose(1, 2).contiguous() for o in old]  # [tiles, 16, hkv, ..]
    for o, x in zip(new, (kc, kp, vc, vp)):
        o[row, pos % BLOCK] = x
    new = [o.transpose(1, 2) for o in new]
    st["cache"][where] = _pack(*new)
    kc, kp, vc, vp = _unpack(st["cache"][where], d)
    ws, wa = _ragged(st["count"], device)
    k_win, v_win = (_values(*z).transpose(1, 2)[begin[ws] + wa // BLOCK, wa % BLOCK].to(BF16) for z in ((kc, kp), (vc, vp)))
    out = [q.flatten(1).to(BF16), k_win, v_win]
    return out + ([k.flatten(1).to(BF16)] if st["fresh"] else [])


# ---- the definition in 64 bits -----------------------------------------------------------------

def _byte(cache, page, tile, head, at):
    return cache[page, tile, head, at].long()


def _read(st, slot, tokens):
    """K and V of the given tokens of one slot in 64 bits [tokens, hkv, D], read nibble by nibble from the cache."""
    d, hkv, page, cache = st["d"], st["hkv"], st["page"], st["cache"]
    w = d // 32
    t = tokens[:, None, None]
    h = torch.arange(hkv, device=cache.device)[None, :, None]
    i = torch.arange(d, device=cache.device)[None, None, :]
    pg, tile, r = st["tables"][slot].long()[t // page], t % page // BLOCK, t % BLOCK
    at_k = 4 * ((r * 4 + i // 8 % 4) * w + i // 32) + i % 8 // 2
    at_v = 9 * d + 4 * ((r // 8 * 32 + i // 4 % 8 * 4 + r % 8 // 2) * w + i // 32) + r % 2 * 2 + i % 4 // 2
    out = []
    for at, pairs in ((at_k, 8 * d), (at_v, 17 * d)):
        code = _byte(cache, pg, tile, h, at) >> (i % 2 * 4) & 15
        p = pairs + 4 * (r * (d // GROUP) + i // GROUP)
        s, m = ((_byte(cache, pg, tile, h, p + o) | _byte(cache, pg, tile, h, p + o + 1) << 8).to(torch.int16).view(BF16).double() for o in (0, 2))
        out.append(code * s + m)
    return out


def _exact_attend(q, k, v, pre, scale):
    """q [R, hq, D], k and v [L, hkv, D] in 64 bits; row r sees the keys up to r + pre."""
    group = q.shape[1] // k.shape[1]
    out = torch.empty_like(q)
    hidden = torch.arange(k.shape[0], device=q.device)[None] > torch.arange(q.shape[0], device=q.device)[:, None] + pre
    for h in range(q.shape[1]):
        s = (q[:, h] @ k[:, h // group].T) * scale
        out[:, h] = torch.softmax(s.masked_fill(hidden, -math.inf), -1) @ v[:, h // group]
    return out


def exact(case, seed):
    st = prepare(case, seed)
    q, pre, hq, hkv, d = st["q"], st["pre"], st["hq"], st["hkv"], st["d"]
    if case["op"] == "prompt":
        parts = zip(st["query"].split(q), st["key"].split(st["k_lens"]), st["value"].split(st["k_lens"]), pre)
        return torch.cat([_exact_attend(a.double(), b.double(), c.double(), p, st["scale"]) for a, b, c, p in parts])
    device = st["cache"].device
    if case["op"] == "cached":
        out = []
        for i, x in enumerate(st["query"].reshape(-1, hq, d).split(q)):
            k, v = (torch.cat(z) for z in zip(*(_read(st, i, t) for t in torch.arange(q[i] + pre[i], device=device).split(4096))))
            out.append(_exact_attend(x.double(), k, v, pre[i], st["scale"]).flatten(1))
        return torch.cat(out)
    outs = [[], [], [], []]
    for i, x in enumerate(st["qkv"].double().split(q)):
        x = x.reshape(-1, hq + 2 * hkv, d)
        pos = torch.arange(pre[i], pre[i] + q[i], device=device)
        angle = st["cos_sin"][pos].double()[:, None]
        turn = torch.complex(angle[..., :d // 2], angle[..., d // 2:])
        z = torch.complex(x[:, :hq + hkv, :d // 2].contiguous(), x[:, :hq + hkv, d // 2:].contiguous()) * turn
        z = torch.cat([z.real, z.imag], -1)
        outs[0].append(z[:, :hq].flatten(1))
        outs[3].append(z[:, hq:].flatten(1))
        for o, y, held in zip(outs[1:3], (z[:, hq:], x[:, hq + hkv:]), _read(st, i, torch.arange(st["start"][i], pre[i], device=device))):
            y = y.reshape(-1, hkv, d // GROUP, GROUP)
            lo, hi = y.min(-1, keepdim=True).values, y.max(-1, keepdim=True).values
            m, s = lo.to(BF16).double(), ((hi - lo) / 15).to(BF16).double()
            code = torch.where(s > 0, torch.round((y - m) / s.clamp_min(1e-300)), torch.zeros_like(y)).clamp(0, 15)
            o.append(torch.cat([held, (code * s + m).reshape(-1, hkv, d)]))
    outs = [torch.cat(o) for o in outs]
    return outs if st["fresh"] else outs[:3]
