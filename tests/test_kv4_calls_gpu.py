"""Forms in which the 4-bit cache and prompt calls take their slots, rows and streams. What is
written is compared with the plain forms entry by entry; attention with 64 bits, under the
bound of tests/test_kv4_gpu.py: an output is rounded to bf16 once (2^-8 of itself), its weights
enter the value product in bf16 (2^-8 of sum p |v|, a 4-bit value counting as |s code| + |m|) and
what else fp32 and fp16 round is below 2^-10 of that sum."""
import pytest
import torch

from tests import kv4_reference as ref

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


def _randn(g, *shape, dtype=BF):
    return torch.randn(*shape, generator=g, device=g.device).to(dtype)


def _gen(dev, seed):
    return torch.Generator(device=dev).manual_seed(seed)


def _cos_sin(n, d, dev):
    a = torch.outer(torch.arange(n, dtype=torch.float64), 10000.0 ** (-torch.arange(0, d, 2, dtype=torch.float64) / d))
    return torch.cat([a.cos(), a.sin()], -1).to(BF).to(dev)


def _near_cached(got, q, cache, table, tokens, scale, what):
    """got, q [rows, hq, D]: attention of the newest rows over `tokens` cached ones of one slot."""
    d = q.shape[-1]
    (_, k), (code, v) = ref.read_cache(cache, table, torch.arange(tokens, device=q.device), d)
    bare = cache.clone()
    bare[..., 9 * d:17 * d] = 0
    low = ref.read_cache(bare, table, torch.arange(tokens, device=q.device), d)[1][1]  # the minima alone
    want = ref.attend_fast(q, k, v, scale)
    mass = ref.attend_fast(q, k, (v - low).abs() + low.abs(), scale)
    got = got.double()
    assert torch.isfinite(got).all(), what
    bound = 2.0 ** -8 * want.abs() + (2.0 ** -8 + 2.0 ** -10) * mass + 1e-30
    worst = ((got - want).abs() / bound).max().item()
    assert worst <= 1.0, f"{what}: {worst:.3g} of the bound"


@pytest.mark.parametrize("d,hq,hkv", [(128, 8, 2), (64, 4, 4)])
@pytest.mark.parametrize("as_rows", [False, True])
@pytest.mark.parametrize("bound", [0, 9000])
def test_tables_and_caches_of_different_sizes(native, cuda, d, hq, hkv, as_rows, bound):
    """Per-slot block tables of different lengths and caches of different page counts: every slot
    reaches its own last page, in all three calls."""
    from swarmlora_b200 import worker_ops as wo
    g = _gen(cuda, d + hq)
    page, ctx, rows = 16, [20, 630, 0, 75], [3, 1, 40, 5]
    per = [2, 40, 3, 5]        # table entries
    pages = [4, 61, 3, 90]     # pages of each slot's cache
    tables, caches = [], []
    for n, m in zip(per, pages):
        # distinct pages, the cache's last one in the table's last entry
        t = torch.randperm(m - 1, generator=g, device=cuda)[:n - 1].to(torch.int32)
        t = torch.cat([t, torch.tensor([m - 1], dtype=torch.int32, device=cuda)])
        tables.append(t)
        caches.append(wo.kv4_cache(m, hkv, d, page, device=cuda))
    for t, c, n in zip(tables, caches, ctx):
        if n:
            ref.write_cache(c, t, torch.arange(n, device=cuda),
                            *(_randn(g, n, hkv, d, dtype=torch.float32) for _ in range(2)))
    qkv = [_randn(g, r, (hq + 2 * hkv) * d) for r in rows]
    cs = _cos_sin(700, d, cuda)
    lens = [torch.tensor([n], dtype=torch.int32, device=cuda) for n in ctx]
    total = [a + b for a, b in zip(ctx, rows)]
    assert all((a - 1) // page == n - 1 for a, n in zip(total, per))  # the last entry holds a new token
    given = [torch.stack([t, t])[:1] for t in tables] if as_rows else tables
    q_rot = torch.empty(sum(rows), hq * d, dtype=BF, device=cuda)
    wo.kv4_append(qkv, given, caches, lens, q_rot, cs, hq, hkv, head_dim=d)
    for i, (x, t, c) in enumerate(zip(qkv, tables, caches)):
        pos = torch.arange(ctx[i], total[i], device=cuda)
        x = x.unflatten(-1, (-1, d))
        new = ref.rotate(x[:, hq:hq + hkv], cs[pos]), x[:, hq + hkv:].float()
        for (code, _), y in zip(ref.read_cache(c, t, pos, d), new):
            _, s, m = ref.quantise(y)
            quot = ((y.unflatten(-1, (-1, 64)).double() - m.double()) / s.double()).clamp(0, 15).flatten(-2)
            # half a step, and what fp32 rounds of the difference and of the quotient: 2^-23 of at most 16
            assert bool(((code - quot).abs() <= 0.5 + 2.0 ** -19).all()), f"slot {i}"
    k_out, v_out = (torch.empty(sum(total), hkv, d, dtype=BF, device=cuda) for _ in range(2))
    wo.kv4_gather(given, caches, [0] * 4, total, k_out, v_out, hkv, head_dim=d)
    for i, (k, v) in enumerate(zip(k_out.split(total), v_out.split(total))):
        for (_, x), got in zip(ref.read_cache(caches[i], tables[i], torch.arange(total[i], device=cuda), d), (k, v)):
            assert torch.equal(got, x.float().to(BF)), f"slot {i}"
    outs = [torch.empty(r, hq * d, dtype=BF, device=cuda) for r in rows]
    wo.paged_attention_kv4(rows, given, caches, lens, outs, q_rot, hq, hkv, max(*total, bound), d ** -0.5, head_dim=d)
    for i, (o, q) in enumerate(zip(outs, q_rot.split(rows))):
        _near_cached(o.view(-1, hq, d), q.reshape(-1, hq, d), caches[i], tables[i], total[i], d ** -0.5, f"slot {i}")


def test_one_size_given_once(native, cuda):
    """The C calls with one table length and page count for all slots write and read what the calls with
    each slot's own do."""
    from swarmlora_b200 import worker_ops as wo
    g = _gen(cuda, 3)
    hq, hkv, d, rows, ctx = 8, 2, 128, [2, 19], [30, 5]
    n, total = len(rows), [a + b for a, b in zip(rows, ctx)]
    tables = torch.randperm(8, generator=g, device=cuda).to(torch.int32).reshape(2, 4)
    lens = torch.tensor(ctx, dtype=torch.int32, device=cuda)
    qkv = _randn(g, sum(rows), (hq + 2 * hkv) * d)
    cs, L, p = _cos_sin(64, d, cuda), native.lib(), native.ptr_array
    stream = torch.cuda.current_stream().cuda_stream
    counts, width = native.i32_array(rows), (hq + 2 * hkv) * d
    tp, lp = p([t.data_ptr() for t in tables]), p([t.data_ptr() for t in lens.split(1)])
    src = p([t.data_ptr() for t in qkv.split(rows)])
    got = []
    for each in (False, True):
        cache = wo.kv4_cache(8, hkv, d, device=cuda)
        q, out = (torch.zeros(sum(rows), hq * d, dtype=BF, device=cuda) for _ in range(2))
        k, v = (torch.zeros(sum(total), hkv, d, dtype=BF, device=cuda) for _ in range(2))
        if each:
            wo.kv4_append(list(qkv.split(rows)), list(tables), cache, lens, q, cs, hq, hkv)
            wo.kv4_gather(list(tables), cache, [0, 0], total, k, v, hkv)
            wo.paged_attention_kv4(rows, list(tables), cache, lens, out, q, hq, hkv, 64, 0.1)
        else:
            cp = p([cache.data_ptr()] * n)
            native.check(L.swl_kv4_append(n, counts, src, width, tp, 4, cp, 8, lp, hq, hkv, d, 16, cs.data_ptr(), 64,
                                          q.data_ptr(), None, stream))
            native.check(L.swl_kv4_gather(n, native.i32_array([0, 0]), native.i32_array(total), tp, 4, cp, 8, hkv, d, 16,
                                          k.data_ptr(), v.data_ptr(), stream))
            native.check(L.swl_paged_attention_kv4(n, counts, tp, 4, cp, 8, lp, p([o.data_ptr() for o in out.split(rows)]),
                                                   hq * d, hq, hkv, d, 16, 0.1, 64, q.data_ptr(), None, stream))
        got.append((cache, q, k, v, out))
    assert all(torch.equal(a, b) for a, b in zip(*got))


def test_packed_rows_beside_listed_tables(native, cuda):
    """Rows packed in one tensor with a list of tables and caches give what all-packed calls give; rows whose elements
    lie apart are refused in both forms, and nothing is written."""
    from swarmlora_b200 import worker_ops as wo
    g = _gen(cuda, 7)
    hq, hkv, d, rows = 4, 2, 128, [3, 1, 20]
    T, width = sum(rows), (hq + 2 * hkv) * d
    tables = torch.arange(12, dtype=torch.int32, device=cuda).reshape(3, 4)
    lens = torch.tensor([9, 0, 30], dtype=torch.int32, device=cuda)
    qkv, cs = _randn(g, T, width + 8)[:, :width], _cos_sin(64, d, cuda)
    res = []
    for listed in (False, True):
        cache = wo.kv4_cache(12, hkv, d, device=cuda)
        q, wide = torch.empty(T, hq * d, dtype=BF, device=cuda), torch.zeros(T, hq * d + 16, dtype=BF, device=cuda)
        out = wide[:, 8:8 + hq * d]
        t, c = (list(tables), [cache] * 3) if listed else (tables, cache)
        wo.kv4_append(qkv, t, c, lens, q, cs, hq, hkv, rows=rows)
        wo.paged_attention_kv4(rows, t, c, lens, out, q, hq, hkv, 64, 0.1)
        apart = torch.zeros(width, T, dtype=BF, device=cuda).t()
        kept = torch.full((hq * d, T), 9.0, dtype=BF, device=cuda)
        with pytest.raises(ValueError, match="qkv"):
            wo.kv4_append(apart, t, c, lens, q, cs, hq, hkv, rows=rows)
        with pytest.raises(ValueError, match="out"):
            wo.paged_attention_kv4(rows, t, c, lens, kept.t(), q, hq, hkv, 64, 0.1)
        assert bool((kept == 9.0).all())
        res.append((cache, q, wide))
    assert all(torch.equal(a, b) for a, b in zip(*res))


def test_attention_under_the_largest_bound(native, cuda):
    from swarmlora_b200 import worker_ops as wo
    g = _gen(cuda, 9)
    hq, hkv, d, rows, ctx = 8, 2, 128, [1, 3, 1], [0, 500, 3000]
    tables = torch.randperm(3 * 190, generator=g, device=cuda).to(torch.int32).reshape(3, 190)
    cache = wo.kv4_cache(3 * 190, hkv, d, device=cuda)
    for t, n in zip(tables, ctx):
        ref.write_cache(cache, t, torch.arange(n + 3, device=cuda),
                        *(_randn(g, n + 3, hkv, d, dtype=torch.float32) for _ in range(2)))
    q, out = _randn(g, sum(rows), hq * d), torch.empty(sum(rows), hq * d, dtype=BF, device=cuda)
    lens = torch.tensor(ctx, dtype=torch.int32, device=cuda)
    wo.paged_attention_kv4(rows, tables, cache, lens, out, q, hq, hkv, 2 ** 31 - 1, d ** -0.5)
    for i, (o, x) in enumerate(zip(out.split(rows), q.split(rows))):
        _near_cached(o.view(-1, hq, d), x.view(-1, hq, d), cache, tables[i], ctx[i] + rows[i], d ** -0.5, f"slot {i}")


@pytest.mark.parametrize("ctx,bound", [(2700, 0), (2700, 9000), (30000, 0)])
@pytest.mark.parametrize("d,hq,hkv,rows", [(128, 8, 2, 1), (128, 16, 2, 1), (64, 8, 2, 1), (64, 16, 2, 1), (128, 8, 2, 4), (64, 8, 2, 4)])
def test_a_flat_tail_behind_one_large_score(native, cuda, ctx, bound, d, hq, hkv, rows):
    """The first key's weight is 2^20 to 2^28 times that of each other key, and its value is 0, so
    the output is the tail's alone. A weight passes through fp16 as 2^7 times itself: below 2^-21 of the
    largest it is off by up to 2^-32 of that, here so much of every token's |s code| + |m|."""
    from swarmlora_b200 import worker_ops as wo
    g = _gen(cuda, ctx + hq)
    n = ctx + rows
    table = torch.randperm(-(-n // 16), generator=g, device=cuda).to(torch.int32)
    cache = wo.kv4_cache(table.numel(), hkv, d, device=cuda)
    k = torch.zeros(n, hkv, d, device=cuda)
    k[0, :, :64] = 1.0
    v = 1.0 + 0.25 * torch.randn(n, hkv, d, generator=g, device=cuda)
    v[0] = 0.0
    ref.write_cache(cache, table, torch.arange(n, device=cuda), k, v)
    powers = torch.tensor([20.0, 24.4, 25.2, 28.0], device=cuda).repeat(hq // 4)
    q = torch.zeros(rows, hq, d, dtype=BF, device=cuda)
    q[..., :64] = (powers * 0.6931471805599453 / 64).to(BF)[:, None]
    out = torch.empty(rows, hq * d, dtype=BF, device=cuda)
    lens = torch.tensor([ctx], dtype=torch.int32, device=cuda)
    wo.paged_attention_kv4([rows], table[None], cache, lens, out, q.flatten(1), hq, hkv, max(n, bound), 1.0, head_dim=d)
    (_, kk), (code, vv) = ref.read_cache(cache, table, torch.arange(n, device=cuda), d)
    bare = cache.clone()
    bare[..., 9 * d:17 * d] = 0
    low = ref.read_cache(bare, table, torch.arange(n, device=cuda), d)[1][1]
    parts = (vv - low).abs() + low.abs()
    want, mass = ref.attend_fast(q, kk, vv, 1.0), ref.attend_fast(q, kk, parts, 1.0)
    lost = 2.0 ** -32 * parts.sum(0).repeat_interleave(hq // hkv, 0)
    off = (out.view(rows, hq, d).double() - want).abs()
    limit = 2.0 ** -8 * want.abs() + (2.0 ** -8 + 2.0 ** -10) * mass + lost
    assert bool((off <= limit).all()), f"{(off / limit).max().item():.3g} of the bound"


@pytest.mark.parametrize("bound", [64, 9000])
def test_slots_without_rows_may_be_empty(native, cuda, bound):
    """Slots that take no part have empty rows, tables and lengths: the others get what they get without them."""
    from swarmlora_b200 import worker_ops as wo
    g = _gen(cuda, 12)
    hq, hkv, d, rows = 4, 2, 128, [0, 3, 0, 1, 0]
    width, cs = (hq + 2 * hkv) * d, _cos_sin(64, d, cuda)
    ints = dict(dtype=torch.int32, device=cuda)
    tables = torch.arange(8, **ints).reshape(2, 4)
    lens = torch.tensor([9, 30], **ints)
    qkv = _randn(g, 4, width)
    want, got = [], []
    for idle, res in ((False, want), (True, got)):
        cache = wo.kv4_cache(8, hkv, d, device=cuda)
        q, out = torch.empty(4, hq * d, dtype=BF, device=cuda), torch.empty(4, hq * d, dtype=BF, device=cuda)
        k, v = (torch.zeros(43, hkv, d, dtype=BF, device=cuda) for _ in range(2))
        if idle:
            nothing = torch.empty(0, **ints)
            spare = wo.kv4_cache(0, hkv, d, device=cuda)
            x, o = ([t[:0], t[:3], t[:0], t[3:], torch.empty(0, t.shape[1], dtype=BF, device=cuda)] for t in (qkv, out))
            t, n = [nothing, tables[0], nothing, tables[1], nothing], [nothing, lens[:1], nothing, lens[1:], nothing]
            c = [spare, cache, spare, cache, spare]
            wo.kv4_append(x, t, c, n, q, cs, hq, hkv)
            wo.kv4_gather(t, c, [0] * 5, [0, 12, 0, 31, 0], k, v, hkv)
            wo.paged_attention_kv4(rows, t, c, n, o, q, hq, hkv, bound, 0.1)
        else:
            wo.kv4_append(qkv, tables, cache, lens, q, cs, hq, hkv, rows=[3, 1])
            wo.kv4_gather(tables, cache, [0, 0], [12, 31], k, v, hkv)
            wo.paged_attention_kv4([3, 1], tables, cache, lens, out, q, hq, hkv, bound, 0.1)
        res += [cache, q, k, v, out]
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    # and a step in which nobody does
    none = torch.empty(0, width, dtype=BF, device=cuda)
    q0, o0 = (torch.empty(0, hq * d, dtype=BF, device=cuda) for _ in range(2))
    k0 = torch.empty(0, hkv, d, dtype=BF, device=cuda)
    for r, t, n in (([0, 0], tables, lens), ([], tables[:0], lens[:0])):
        wo.kv4_append(none, t, want[0], n, q0, cs, hq, hkv, rows=r)
        wo.kv4_gather(t, want[0], r, r, k0, k0, hkv)
        wo.paged_attention_kv4(r, t, want[0], n, o0, q0, hq, hkv, bound, 0.1)
    torch.cuda.synchronize()
    assert torch.equal(want[0], got[0])


def test_a_call_on_a_stream_of_its_own(native, cuda):
    """Each call on a side stream, made by torch or wrapped from its handle."""
    from swarmlora_b200 import worker_ops as wo
    g = _gen(cuda, 14)
    hq, hkv, d, rows = 4, 2, 128, [3, 20]
    T, cs = sum(rows), _cos_sin(64, d, cuda)
    tables = torch.arange(8, dtype=torch.int32, device=cuda).reshape(2, 4)
    lens, qkv = torch.tensor([9, 30], dtype=torch.int32, device=cuda), _randn(g, T, (hq + 2 * hkv) * d)
    side = torch.cuda.Stream()
    res = []
    for stream in (None, side, torch.cuda.ExternalStream(side.cuda_stream)):
        cache = wo.kv4_cache(8, hkv, d, device=cuda)
        q, out = (torch.zeros(T, hq * d, dtype=BF, device=cuda) for _ in range(2))
        k, v = (torch.zeros(62, hkv, d, dtype=BF, device=cuda) for _ in range(2))
        torch.cuda.synchronize()
        wo.kv4_append(qkv, tables, cache, lens, q, cs, hq, hkv, rows=rows, stream=stream)
        wo.kv4_gather(tables, cache, [0, 0], [12, 50], k, v, hkv, stream=stream)
        wo.paged_attention_kv4(rows, tables, cache, lens, out, q, hq, hkv, 64, 0.1, stream=stream)
        o = wo.prompt_attention(q.view(T, hq, d), k, v, rows, [12, 50], stream=stream)
        torch.cuda.synchronize()
        res.append((cache, q, k, v, out, o))
    assert all(torch.equal(a, b) and torch.equal(a, c) for a, b, c in zip(*res))


def test_no_wait_ran_out(native, cuda):
    from swarmlora_b200 import worker_ops as wo
    assert wo.attention_device_error() == 0 and wo.attention_device_error(cuda) == 0


def _check_plan(dev, rows, ctx, hq, hkv, d, bound, whole, seed):
    """Attention of slots over one cache whose unused tokens are NaN, under a bound whose plan is asserted."""
    from swarmlora_b200 import worker_ops as wo
    assert (wo.kv4_part_floats(rows, hq, hkv, bound, head_dim=d) == 0) == whole
    g = _gen(dev, seed)
    per = -(-max(a + b for a, b in zip(rows, ctx)) // 16)
    tables = torch.randperm(len(rows) * per + 2, generator=g, device=dev)[:len(rows) * per].to(torch.int32).reshape(-1, per)
    cache = torch.full((tables.numel() + 2, 1, hkv, 18 * d), 0xff, dtype=torch.uint8, device=dev)
    for t, r, n in zip(tables, rows, ctx):
        ref.write_cache(cache, t, torch.arange(n + r, device=dev),
                        *(_randn(g, n + r, hkv, d, dtype=torch.float32) for _ in range(2)))
    q = _randn(g, sum(rows), hq * d)
    out = torch.full((sum(rows) + 1, hq * d), 9.0, dtype=BF, device=dev)
    wo.paged_attention_kv4(rows, tables, cache, torch.tensor(ctx, dtype=torch.int32, device=dev), out, q, hq, hkv, bound,
                           d ** -0.5, head_dim=d)
    assert bool((out[sum(rows):] == 9.0).all())
    for i, (o, x) in enumerate(zip(out[:sum(rows)].split(rows), q.split(rows))):
        if rows[i]:
            _near_cached(o.view(-1, hq, d), x.view(-1, hq, d), cache, tables[i], ctx[i] + rows[i], d ** -0.5,
                         f"slot {i} of {rows}/{ctx}")


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("hq,hkv", [(8, 2), (10, 2), (16, 2), (24, 4)])  # groups of 4 (blocks in pairs), 5, 8 and 6
@pytest.mark.parametrize("ctx,bound,whole", [
    ([0, 40, 126], 127, True), ([127], 128, True), ([128, 0, 63], 129, True),  # four warps up to 128 tokens, six beyond
    ([1007, 1000], 1008, True), ([2800, 1, 2750], 2801, True), ([2815], 2816, True),
    ([2816, 2799, 15], 2817, False), ([3000, 100], 3100, False), ([128, 5], 2817, False)])
def test_single_rows_on_both_sides_of_each_plan(native, cuda, d, hq, hkv, ctx, bound, whole):
    _check_plan(cuda, [1] * len(ctx), ctx, hq, hkv, d, bound, whole, seed=sum(ctx) + hq)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("rows,ctx,hq,hkv,bound,whole", [
    ([2, 1, 2], [500, 2700, 0], 8, 2, 2816, True), ([1, 2], [2814, 2815], 8, 2, 2817, False),       # one column tile
    ([4, 0, 1, 9], [2900, 5, 31, 4], 8, 2, 2904, True), ([3, 5], [5000, 100], 8, 2, 5120, True),     # two
    ([3, 5], [5118, 5115], 8, 2, 5121, False), ([7, 1], [900, 130], 6, 6, 5121, False),
    ([1] * 60, [36 * i for i in range(60)], 32, 8, 2176, True),                                      # many pairs
    ([1] * 60, [36 * i for i in range(60)], 32, 8, 2177, False),
    ([5, 4, 3, 2, 1] * 6, [70 * i for i in range(30)], 32, 8, 2176, True)])
def test_several_rows_on_both_sides_of_each_plan(native, cuda, d, rows, ctx, hq, hkv, bound, whole):
    _check_plan(cuda, rows, ctx, hq, hkv, d, bound, whole, seed=sum(ctx) + sum(rows))


@pytest.mark.parametrize("d,hkv", [(64, 3), (128, 2)])
def test_codes_are_those_of_ieee_quotients(native, cuda, d, hkv):
    """Codes of groups of all scales and offsets, bit for bit: fp32 difference, fp32 quotient, nearest even, within 0 .. 15.
    (Angles of 0: k is quantised as it stands.)"""
    from swarmlora_b200 import worker_ops as wo
    g = torch.Generator().manual_seed(d)
    T = 4096
    x = torch.randn(T, 2 * hkv, d // 64, 64, generator=g)
    up = torch.exp2(torch.randint(-120, 100, (T, 2 * hkv, d // 64, 1), generator=g).float())
    offset = torch.randn(T, 2 * hkv, d // 64, 1, generator=g) * torch.exp2(torch.randint(-8, 8, up.shape, generator=g).float())
    x[::3] = x[::3].mul(8).round().div(8)     # many quotients on or next to the middle between two codes
    x[1::3] = torch.randint(0, 31, x[1::3].shape, generator=g).float() / 2
    rows = ((x + offset) * up).to(BF).reshape(T, -1)
    page = 1024
    tables = torch.randperm(4, generator=g).to(torch.int32)[None].to(cuda)
    cache = wo.kv4_cache(4, hkv, d, page, device=cuda)
    qkv = torch.cat([torch.zeros(T, d, dtype=BF), rows], 1).to(cuda)
    cs = torch.cat([torch.ones(T, d // 2), torch.zeros(T, d // 2)], 1).to(BF).to(cuda)
    q_rot = torch.empty(T, d, dtype=BF, device=cuda)
    wo.kv4_append(qkv, tables, cache, torch.zeros(1, dtype=torch.int32, device=cuda), q_rot, cs, 1, hkv, head_dim=d, page=page,
                  rows=[T])
    got = ref.read_cache(cache.cpu(), tables[0].cpu(), torch.arange(T), d)
    for (code, _), y in zip(got, rows.float().reshape(T, 2, hkv, d).unbind(1)):
        y = y.unflatten(-1, (-1, 64))
        _, s, m = ref.quantise(y.flatten(-2))
        quot = torch.where(s.float() > 0, (y - m.float()) / s.float(), torch.zeros(()))
        want = quot.round().clamp(0, 15).long().flatten(-2)
        assert torch.equal(code, want), int((code != want).sum())


@pytest.mark.parametrize("rows,hq,hkv,d", [([1, 1], 8, 2, 128), ([3, 1], 8, 2, 64), ([4, 20], 16, 2, 128)])
@pytest.mark.parametrize("bound", [290, 3000, 5300])
def test_contexts_beyond_the_bound_are_cut_there(native, cuda, rows, hq, hkv, d, bound):
    """A row at or behind max_len sees the first max_len tokens."""
    from swarmlora_b200 import worker_ops as wo
    g = _gen(cuda, bound)
    ctx, n = [bound + 130, bound - 2], -(-(bound + 200) // 16)
    tables = torch.randperm(2 * n, generator=g, device=cuda).to(torch.int32).reshape(2, n)
    cache = wo.kv4_cache(2 * n, hkv, d, device=cuda)
    for t in tables:
        ref.write_cache(cache, t, torch.arange(16 * n, device=cuda),
                        *(_randn(g, 16 * n, hkv, d, dtype=torch.float32) for _ in range(2)))
    q, out = _randn(g, sum(rows), hq * d), torch.empty(sum(rows), hq * d, dtype=BF, device=cuda)
    wo.paged_attention_kv4(rows, tables, cache, torch.tensor(ctx, dtype=torch.int32, device=cuda), out, q, hq, hkv, bound,
                           d ** -0.5, head_dim=d)
    at = 0
    for i, r in enumerate(rows):
        for j in range(r):
            _near_cached(out[at].view(1, hq, d), q[at].view(1, hq, d), cache, tables[i], min(ctx[i] + j + 1, bound),
                         d ** -0.5, f"row {j} of slot {i}")
            at += 1


@pytest.mark.parametrize("bound", [64, 9000])
def test_slots_of_negative_length(native, cuda, bound):
    """Positions below 0 are not cached and see nothing; rows that reach position 0 count from there."""
    from swarmlora_b200 import worker_ops as wo
    g = _gen(cuda, 16)
    hq, hkv, d, rows, ctx = 4, 2, 128, [2, 4, 1], [-100, -2, -(2 ** 31)]
    tables = torch.tensor([[0], [1], [2]], dtype=torch.int32, device=cuda)
    cache = torch.full((3, 1, hkv, 18 * d), 0x11, dtype=torch.uint8, device=cuda)
    before = cache.clone()
    lens, qkv = torch.tensor(ctx, dtype=torch.int32, device=cuda), _randn(g, 7, (hq + 2 * hkv) * d)
    q, out = (torch.full((7, hq * d), 9.0, dtype=BF, device=cuda) for _ in range(2))
    wo.kv4_append(qkv, tables, cache, lens, q, _cos_sin(64, d, cuda), hq, hkv, rows=rows)
    hidden = [0, 1, 2, 3, 6]
    assert bool((q[hidden] == 0).all()) and bool((q[[4, 5]] != 0).any())
    assert torch.equal(cache[[0, 2]], before[[0, 2]]) and not torch.equal(cache[1], before[1])
    wo.paged_attention_kv4(rows, tables, cache, lens, out, q, hq, hkv, bound, 0.1)
    assert bool((out[hidden] == 0).all())
    for r, n in ((4, 1), (5, 2)):
        _near_cached(out[r].view(1, hq, d), q[r].view(1, hq, d), cache, tables[1], n, 0.1, f"row {r}")


@pytest.mark.parametrize("bound,whole", [(1000, True), (2817, False)])
def test_as_many_slots_as_a_call_takes(native, cuda, bound, whole):
    """128 slots of one to three rows, some without any."""
    rows = [(i % 4) for i in range(128)]
    _check_plan(cuda, rows, [(37 * i) % 400 for i in range(128)], 4, 2, 64, bound, whole, seed=128)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("group", [3, 17, 33, 64, 65, 100, 127, 128])
def test_prompts_of_many_query_heads_a_kv_head(native, cuda, d, group):
    """Tiles that no token count fills exactly, down to one token a tile."""
    from swarmlora_b200 import worker_ops as wo
    g = _gen(cuda, group + d)
    hkv = 2
    q_lens, k_lens = [1, 5, 40, 0, 3], [300, 5, 170, 2, 1]
    q, k, v = (_randn(g, sum(n), h, d) for n, h in ((q_lens, hkv * group), (k_lens, hkv), (k_lens, hkv)))
    out = torch.full((sum(q_lens) + 2, hkv * group, d), 9.0, dtype=BF, device=cuda)
    wo.prompt_attention(torch.cat([q, q[:2]]), k, v, q_lens, k_lens, out=out)
    assert bool((out[sum(q_lens):] == 9.0).all())
    for a, b, c, o in zip(q.split(q_lens), k.split(k_lens), v.split(k_lens), out.split([*q_lens, 2])):
        want, mass = (ref.attend_fast(a, b, x, d ** -0.5) for x in (c, c.abs()))
        off = (o.double() - want).abs()
        assert bool((off <= 2.0 ** -8 * want.abs() + (2.0 ** -8 + 2.0 ** -10) * mass + 1e-30).all())
    assert wo.attention_device_error() == 0


@pytest.mark.parametrize("hq,rows", [(8, 1), (16, 1), (16, 3)])
@pytest.mark.parametrize("power", [0, 20, 22, 23, 24, 25])
def test_weights_of_huge_scores_stay_finite(native, cuda, hq, rows, power):
    """Scores around -2^power (base 2), each of a warp's block pairs 9.4 above the last: next to 2^8, by which
    a score may pass its reference before that moves. fp32 holds such scores to steps of up to 4, so
    only what they cannot change is looked at: values of 1 have 1 as every weighted mean, up to the fp16 rounding of a weight (2^-11) and
    the output's (2^-8)."""
    from swarmlora_b200 import worker_ops as wo
    hkv, d, n = 2, 128, 2800
    warps = 6 if rows * hq // hkv <= 8 else 4
    table = torch.arange(n // 16, dtype=torch.int32, device=cuda)
    cache = wo.kv4_cache(n // 16, hkv, d, device=cuda)
    step = torch.arange(n, device=cuda) // 32 // warps
    k = torch.ones(n, hkv, d, device=cuda)
    k[:, :, 64:] = (6.5 * step.clamp(max=19))[:, None, None]
    ref.write_cache(cache, table, torch.arange(n, device=cuda), k, torch.ones(n, hkv, d, device=cuda))
    for i in range(16):
        q = torch.zeros(rows, hq, d, dtype=BF, device=cuda)
        spread = 1.0 + (torch.arange(rows * hq, device=cuda).view(rows, hq) + i * rows * hq) % 128 / 128
        q[..., :64] = (-spread * 2.0 ** power * 0.6931471805599453 / 64).to(BF)[..., None]
        q[..., 64:] = 1.0 / 64
        out = torch.empty(rows, hq * d, dtype=BF, device=cuda)
        wo.paged_attention_kv4([rows], table[None], cache, torch.tensor([n - rows], dtype=torch.int32, device=cuda), out,
                               q.flatten(1), hq, hkv, n, 1.0)
        assert bool(((out.float() - 1.0).abs() <= 2.0 ** -8 + 2.0 ** -11).all()), out.float().sub(1).abs().max().item()


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("rows,ctx", [([1], [4000]), ([1, 1, 1], [40, 0, 3100]), ([3, 0, 1, 16], [2900, 7, 0, 333]), ([1] * 60, [5] * 60)])
def test_what_scratch_holds_beforehand_does_not_matter(native, cuda, d, rows, ctx):
    from swarmlora_b200 import worker_ops as wo
    g = _gen(cuda, sum(ctx))
    hq, hkv, total = 8, 2, [a + b for a, b in zip(rows, ctx)]
    per = -(-max(total) // 16)
    tables = torch.arange(len(rows) * per, dtype=torch.int32, device=cuda).reshape(-1, per)
    cache = wo.kv4_cache(tables.numel(), hkv, d, device=cuda)
    for t, n in zip(tables, total):
        ref.write_cache(cache, t, torch.arange(n, device=cuda), *(_randn(g, n, hkv, d, dtype=torch.float32) for _ in range(2)))
    q, lens = _randn(g, sum(rows), hq * d), torch.tensor(ctx, dtype=torch.int32, device=cuda)
    need = wo.kv4_part_floats(rows, hq, hkv, 6000, head_dim=d)
    assert need > 0
    outs = []
    for fill in (0.0, float("nan")):
        part = torch.full((need,), fill, device=cuda)
        outs.append(torch.full((sum(rows), hq * d), 9.0, dtype=BF, device=cuda))
        wo.paged_attention_kv4(rows, tables, cache, lens, outs[-1], q, hq, hkv, 6000, d ** -0.5, head_dim=d, part=part)
    assert bool(torch.isfinite(outs[0]).all()) and torch.equal(*outs)
