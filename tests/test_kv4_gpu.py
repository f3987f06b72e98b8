"""Prompt attention and the 4-bit cache on the GPU against plain 64-bit forms.

Tolerances count roundings. An attention output is rounded to bf16 once (2^-8 of
itself); the weights enter the value product in bf16 (2^-8 of sum p |v|, where a
4-bit value counts as |s code| + |m|, the two parts it is summed from). What fp32
sums, the exponential and (4-bit cache) the fp16 exchange of the weights add is below
2^-10 of sum p |v| altogether."""
import pytest
import torch

from tests import kv4_reference as ref

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


def _randn(g, *shape, dtype=BF):
    return torch.randn(*shape, generator=g, device=g.device).to(dtype)


def _gen(dev, seed):
    return torch.Generator(device=dev).manual_seed(seed)


def _near(got, want, mass, what, slack=2.0 ** -8 + 2.0 ** -10):
    got = got.double()
    assert torch.isfinite(got).all(), f"{what}: non-finite"
    off = (got - want).abs()
    bound = 2.0 ** -8 * want.abs() + slack * mass + 1e-30
    worst = (off / bound).max().item() if off.numel() else 0.0
    assert worst <= 1.0, f"{what}: {worst:.3g} of the bound"


# ---- whole prompts -------------------------------------------------------------------------------
def _check_prompt(dev, q_lens, k_lens, hq, hkv, d, seed=0, gain=1.0, bias=0.0, fused=False, split_v=True):
    from swarmlora_b200 import worker_ops as wo
    g = _gen(dev, seed)
    tq, tk = sum(q_lens), sum(k_lens)
    q = _randn(g, tq, hq, d) * gain
    if fused:  # views of one projection's rows
        rows = _randn(g, tk, (hq + 2 * hkv) * d)
        k, v = (rows[:, o:o + hkv * d].unflatten(-1, (hkv, d)) for o in (hq * d, (hq + hkv) * d))
    else:
        k, v = _randn(g, tk, hkv, d), _randn(g, tk, hkv, d) + bias
    scale = d ** -0.5
    got = wo.prompt_attention(q, k, v, q_lens, k_lens, scale=scale)
    for i, (a, b, c, o) in enumerate(zip(q.split(q_lens), k.split(k_lens), v.split(k_lens), got.split(q_lens))):
        _near(o, ref.attend_fast(a, b, c, scale), ref.attend_fast(a, b, c.abs(), scale), f"sequence {i} of {q_lens}/{k_lens}")
    return got


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("hq,hkv", [(4, 1), (8, 8), (6, 2), (5, 1), (16, 2), (14, 2)])
def test_prompts_of_all_small_lengths(native, cuda, d, hq, hkv):
    lens = [1, 2, 15, 16, 17, 31, 33, 63, 64, 65, 127, 128, 129, 0, 200, 3]
    _check_prompt(cuda, lens, lens, hq, hkv, d, seed=d + hq)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("q_lens,k_lens", [
    ([1], [1]), ([1], [127]), ([1], [128]), ([1], [129]), ([1], [4097]), ([16], [800]), ([5, 16, 1], [700, 17, 640]),
    ([300], [1000]), ([257, 3], [513, 1030]), ([64, 64], [64, 1200]), ([33], [32 + 129])])
def test_chunks_behind_a_prefix(native, cuda, d, q_lens, k_lens):
    _check_prompt(cuda, q_lens, k_lens, 8, 2, d, seed=sum(k_lens))


@pytest.mark.parametrize("q_lens,k_lens", [([5], [0]), ([9, 4, 7], [3, 0, 7]), ([300, 2], [130, 1]), ([40], [1])])
def test_rows_that_see_no_key_give_zeros(native, cuda, q_lens, k_lens):
    from swarmlora_b200 import worker_ops as wo
    g = _gen(cuda, 3)
    q, k, v = (_randn(g, sum(n), h, 128) for n, h in ((q_lens, 8), (k_lens, 2), (k_lens, 2)))
    got = wo.prompt_attention(q, k, v, q_lens, k_lens)
    for a, b, c, o in zip(q.split(q_lens), k.split(k_lens), v.split(k_lens), got.split(q_lens)):
        none = max(0, a.shape[0] - b.shape[0])
        assert torch.equal(o[:none], torch.zeros_like(o[:none]))
        _near(o, ref.attend_fast(a, b, c, 128 ** -0.5), ref.attend_fast(a, b, c.abs(), 128 ** -0.5), "rows")


def test_fused_rows_and_large_scores(native, cuda):
    _check_prompt(cuda, [130, 77, 1], [130, 77, 1], 8, 2, 128, seed=5, fused=True)
    _check_prompt(cuda, [700], [700], 4, 1, 128, seed=6, gain=30.0)   # scores to +-100: one key takes a row
    _check_prompt(cuda, [513], [900], 4, 2, 64, seed=7, bias=100.0)


def test_long_prompts(native, cuda):
    _check_prompt(cuda, [4099], [4099], 4, 1, 128, seed=8)
    _check_prompt(cuda, [1500, 1, 2049], [1500, 3000, 2049], 4, 4, 64, seed=9)


def test_scores_that_rise_along_the_keys(native, cuda):
    """Every later key scores higher, by more than any one rescale can skip: the running
    maximum moves in every tile."""
    from swarmlora_b200 import worker_ops as wo
    d, n = 128, 1100
    q = torch.zeros(n, 4, d, dtype=BF, device=cuda)
    q[..., 0] = 1.0
    k = torch.zeros(n, 1, d, dtype=BF, device=cuda)
    k[:, 0, 0] = torch.arange(n, device=cuda).to(BF)
    v = _randn(_gen(cuda, 1), n, 1, d)
    for sign in (1, -1):
        got = wo.prompt_attention(q * sign, k, v, [n], scale=1.0)
        _near(got, ref.attend_fast(q * sign, k, v, 1.0), ref.attend_fast(q * sign, k, v.abs(), 1.0), f"sign {sign}")


def test_prompt_values_that_no_row_sees_do_not_matter(native, cuda):
    """NaN and infinity in keys and values behind a row's own position, in the next
    sequence, and behind the last one: rows ahead of them keep their values, and what is
    behind the last sequence is not written."""
    from swarmlora_b200 import worker_ops as wo
    g = _gen(cuda, 11)
    for d in (64, 128):
        lens = [70, 150, 33]
        T = sum(lens)
        q, k, v = _randn(g, T + 5, 8, d), _randn(g, T + 9, 2, d), _randn(g, T + 9, 2, d)
        want = wo.prompt_attention(q[:T], k[:T], v[:T], lens)
        for bad in (float("nan"), float("inf"), -float("inf")):
            k2, v2 = k.clone(), v.clone()
            k2[T:], v2[T:] = bad, bad
            for at in (40, 70 + 100, 70 + 149, T - 1):  # from these rows on, their sequence may differ
                k2[at, 0], v2[at, :, 3] = bad, bad
            out = torch.full((T + 5, 8, d), 7.0, dtype=BF, device=cuda)
            got = wo.prompt_attention(q, k2, v2, lens, out=out)
            assert got is out and bool((out[T:] == 7.0).all())
            clean = torch.ones(T, dtype=torch.bool, device=cuda)
            for lo, hi in ((40, 70), (170, 220), (T - 1, T)):
                clean[lo:hi] = False
            assert torch.equal(out[:T][clean], want[clean]), f"d {d}, {bad}"
            rest = out[:T][~clean].float()
            # a value that is seen shows: dimension 3 of every later row of its sequence
            assert not torch.isfinite(rest[:, 4:, 3]).any()
            assert torch.isfinite(rest[:, 4:, 4:]).all()


def test_prompt_device_stream_and_graph(native, cuda):
    from swarmlora_b200 import worker_ops as wo
    g = _gen(cuda, 12)
    q, k, v = _randn(g, 100, 8, 128), _randn(g, 400, 2, 128), _randn(g, 400, 2, 128)
    want = wo.prompt_attention(q, k, v, [60, 40], [60, 340])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = wo.prompt_attention(q, k, v, [60, 40], [60, 340], stream=side)
    side.synchronize()
    assert torch.equal(got, want)
    graph, out = torch.cuda.CUDAGraph(), torch.empty_like(q)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        wo.prompt_attention(q, k, v, [60, 40], [60, 340], out=out)
    for seed in (1, 2):
        v.copy_(_randn(_gen(cuda, seed), 400, 2, 128))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, wo.prompt_attention(q, k, v, [60, 40], [60, 340]))


# ---- the 4-bit cache -----------------------------------------------------------------------------
def _cos_sin(n, d, dev):
    a = torch.outer(torch.arange(n, dtype=torch.float64), 10000.0 ** (-torch.arange(0, d, 2, dtype=torch.float64) / d))
    return torch.cat([a.cos(), a.sin()], -1).to(BF).to(dev)


def _tables(g, n, per, spare=2):
    return torch.randperm(n * per + spare, generator=g, device=g.device)[:n * per].to(torch.int32).reshape(n, per)


APPEND = [([1], [0]), ([1], [15]), ([1, 1, 1], [16, 31, 500]), ([2], [15]), ([17], [15]), ([40, 1, 0, 33], [0, 7, 3, 63]),
          ([128], [5]), ([300, 16], [1, 32]), ([3, 5, 2], [30, 14, 0])]


@pytest.mark.parametrize("rows,ctx", APPEND)
@pytest.mark.parametrize("d,hq,hkv,page", [(128, 8, 2, 16), (64, 3, 1, 32), (64, 6, 3, 16), (128, 5, 5, 64)])
def test_append_writes_the_definition(native, cuda, rows, ctx, d, hq, hkv, page):
    from swarmlora_b200 import worker_ops as wo
    g = _gen(cuda, sum(rows) + d)
    n, total = len(rows), sum(rows)
    longest = max(a + b for a, b in zip(rows, ctx))
    tables = _tables(g, n, -(-longest // page))
    cache = torch.randint(0, 256, (tables.numel() + 2, page // 16, hkv, 18 * d), generator=g, device=cuda, dtype=torch.uint8)
    before = cache.clone()
    qkv = _randn(g, total, (hq + 2 * hkv) * d + 16)  # a longer row stride
    qkv[:, (hq + hkv) * d:] *= 3.0
    cs = _cos_sin(longest + 3, d, cuda)
    lens = torch.tensor(ctx, dtype=torch.int32, device=cuda)
    q_rot = torch.full((total, hq * d), 9.0, dtype=BF, device=cuda)
    k_rot = torch.full((total, hkv * d), 9.0, dtype=BF, device=cuda)
    wo.kv4_append(qkv, tables, cache, lens, q_rot, cs, hq, hkv, head_dim=d, page=page, rows=rows, k_rot=k_rot)
    expect = before.clone()
    at = 0
    for i, r in enumerate(rows):
        x = qkv[at:at + r, :(hq + 2 * hkv) * d].unflatten(-1, (-1, d))
        pos = torch.arange(ctx[i], ctx[i] + r, device=cuda)
        turned = ref.rotate(x[:, :hq + hkv], cs[pos])
        assert torch.equal(q_rot[at:at + r], turned[:, :hq].flatten(1).to(BF))
        assert torch.equal(k_rot[at:at + r], turned[:, hq:].flatten(1).to(BF))
        k, v = turned[:, hq:], x[:, hq + hkv:].float()
        if r:
            ref.write_cache(expect, tables[i], pos, k, v)
            for (code, _), y in zip(ref.read_cache(cache, tables[i], pos, d), (k, v)):
                # codes: within half a step of the exact quotient, up to the division's own roundings
                _, s, m = ref.quantise(y)
                quot = ((y.unflatten(-1, (-1, 64)).double() - m.double()) / s.double()).clamp(0, 15).flatten(-2)
                assert bool(((code - quot).abs() <= 0.5 + 2.0 ** -18).all())
        at += r
    # everything but a code at a rounding border is as expected, neighbours and other pages included
    differ = cache != expect
    assert int(differ.sum()) <= 2 + total * hkv * d // 20000, int(differ.sum())
    for i, r in enumerate(rows):
        pos = torch.arange(0, ctx[i], device=cuda)
        if ctx[i]:
            assert all(torch.equal(a[0], b[0]) for a, b in zip(ref.read_cache(cache, tables[i], pos, d),
                                                               ref.read_cache(before, tables[i], pos, d)))


def test_append_lists_and_slots_with_their_own_caches(native, cuda):
    """Lists of per-slot tensors give what packed tensors give."""
    from swarmlora_b200 import worker_ops as wo
    g = _gen(cuda, 4)
    rows, ctx, hq, hkv, d, page = [3, 1, 20], [9, 0, 30], 4, 2, 128, 16
    qkv = _randn(g, sum(rows), (hq + 2 * hkv) * d)
    tables = _tables(g, 3, 4, 0)
    cs = _cos_sin(64, d, cuda)
    lens = torch.tensor(ctx, dtype=torch.int32, device=cuda)
    one = wo.kv4_cache(12, hkv, d, page, device=cuda)
    q1, q2 = (torch.empty(sum(rows), hq * d, dtype=BF, device=cuda) for _ in range(2))
    wo.kv4_append(qkv, tables, one, lens, q1, cs, hq, hkv, rows=rows)
    many = [wo.kv4_cache(12, hkv, d, page, device=cuda) for _ in rows]
    wo.kv4_append([t.clone() for t in qkv.split(rows)], [t.clone() for t in tables], many, list(lens.split(1)), q2, cs, hq, hkv)
    assert torch.equal(q1, q2)
    assert torch.equal(one, sum(m.int() for m in many).to(torch.uint8))
    outs = [torch.empty(r, hq * d, dtype=BF, device=cuda) for r in rows]
    flat = torch.empty(sum(rows), hq * d, dtype=BF, device=cuda)
    wo.paged_attention_kv4(rows, tables, one, lens, flat, q1, hq, hkv, 64, 0.1)
    wo.paged_attention_kv4(rows, [t.clone() for t in tables], many, list(lens.split(1)), outs, q1, hq, hkv, 64, 0.1)
    assert torch.equal(torch.cat(outs), flat)


def test_append_groups_of_special_values(native, cuda):
    """Constant groups, groups with a NaN or an infinity, zeros and extremes."""
    from swarmlora_b200 import worker_ops as wo
    hq, hkv, d = 1, 1, 128
    v = torch.randn(8, d, generator=_gen(cuda, 2), device=cuda)
    v[0] = 0.0
    v[1] = -3.25
    v[2, 5] = float("nan")
    v[3, 70] = float("inf")
    v[4, 1] = -float("inf")
    v[5] *= 1e-38
    v[6] *= 1e36
    v[7, :64] = 1e-30
    qkv = torch.zeros(8, 3 * d, dtype=BF, device=cuda)
    qkv[:, 2 * d:] = v.to(BF)
    tables = torch.zeros(1, 1, dtype=torch.int32, device=cuda)
    cache = wo.kv4_cache(1, hkv, d, device=cuda)
    q_rot = torch.empty(8, d, dtype=BF, device=cuda)
    wo.kv4_append(qkv, tables, cache, torch.zeros(1, dtype=torch.int32, device=cuda), q_rot, _cos_sin(16, d, cuda), hq, hkv,
                  rows=[8])
    k_out, v_out = (torch.empty(8, 1, d, dtype=BF, device=cuda) for _ in range(2))
    wo.kv4_gather(tables, cache, [0], [8], k_out, v_out, hkv)
    got, want = v_out[:, 0].float(), qkv[:, 2 * d:].float()
    assert bool((k_out == 0).all())
    assert torch.equal(got[:2], want[:2])
    assert got[2, :64].isnan().all() and got[3, 64:].isnan().all() and got[4, :64].isnan().all()
    for r, side in ((2, slice(64, 128)), (3, slice(0, 64)), (4, slice(64, 128)), (6, slice(0, 128))):
        span = want[r, side].max() - want[r, side].min()
        assert bool(((got[r, side] - want[r, side]).abs() <= span / 30 + 2.0 ** -6 * want[r, side].abs().max()).all())
    assert torch.equal(got[7, :64], want[7, :64])
    assert torch.isfinite(got[5]).all()


def test_positions_and_pages_outside_are_left_alone(native, cuda):
    """Rows past the block table, past the angles or on a page that does not exist write
    nothing, a gather of such pages gives zeros, attention leaves their tokens out."""
    from swarmlora_b200 import worker_ops as wo
    g = _gen(cuda, 21)
    hq, hkv, d = 4, 2, 128
    tables = torch.tensor([[0, 1], [2, 99], [-1, 3], [4, 5]], dtype=torch.int32, device=cuda)
    lens = torch.tensor([30, 14, 14, 20], dtype=torch.int32, device=cuda)
    rows = [4, 4, 4, 4]
    qkv = _randn(g, 16, (hq + 2 * hkv) * d)
    cs = _cos_sin(22, d, cuda)  # positions from 22 on have no angle
    cache = torch.full((6, 1, hkv, 18 * d), 0x11, dtype=torch.uint8, device=cuda)
    before = cache.clone()
    q_rot = torch.full((16, hq * d), 9.0, dtype=BF, device=cuda)
    wo.kv4_append(qkv, tables, cache, lens, q_rot, cs, hq, hkv, rows=rows)
    assert bool((q_rot[:4] == 0).all()) and bool((q_rot[14:] == 0).all()) and bool((q_rot[4:14] != 9.0).any(-1).all())
    same = [bool(torch.equal(cache[p], before[p])) for p in range(6)]
    # slot 0: beyond the angles; slot 1: two rows on page 2, two on no page; slot 2: two on no page, two on page 3;
    # slot 3: positions 20, 21 on page 5
    assert same == [True, True, False, False, True, False]
    k_out, v_out = (torch.full((32, hkv, d), 9.0, dtype=BF, device=cuda) for _ in range(2))
    wo.kv4_gather(tables[1:2], cache, [0], [32], k_out, v_out, hkv)
    assert bool((k_out[16:] == 0).all()) and bool((v_out[16:] == 0).all()) and bool((k_out[14:16] != 9.0).any())
    out = torch.empty(4, hq * d, dtype=BF, device=cuda)
    cache = wo.kv4_cache(6, hkv, d, device=cuda)
    tok = torch.arange(16, device=cuda)
    ref.write_cache(cache, tables[1], tok, *(_randn(g, 16, hkv, d, dtype=torch.float32) for _ in range(2)))
    q = _randn(g, 4, hq * d)
    wo.paged_attention_kv4([4], tables[1:2], cache, torch.tensor([20], dtype=torch.int32, device=cuda), out, q, hq, hkv, 64, 0.1)
    (_, k), (_, v) = ref.read_cache(cache, tables[1], tok, d)
    # every row sees positions 0..15 (the others lie on no page)
    for r in range(4):
        _near(out[r].reshape(1, hq, d), ref.attend_fast(q[r].reshape(1, hq, d), k, v, 0.1),
              ref.attend_fast(q[r].reshape(1, hq, d), k, v.abs() + 8.0, 0.1), f"row {r}")
    # a slot none of whose pages exist gives zeros
    none = torch.full((1, 2), -5, dtype=torch.int32, device=cuda)
    out.fill_(9.0)
    wo.paged_attention_kv4([4], none, cache, torch.tensor([20], dtype=torch.int32, device=cuda), out, q, hq, hkv, 64, 0.1)
    assert bool((out == 0).all())


@pytest.mark.parametrize("d,hkv,page", [(128, 2, 16), (64, 3, 64), (128, 8, 32)])
def test_gather_reads_any_range(native, cuda, d, hkv, page):
    from swarmlora_b200 import worker_ops as wo
    g = _gen(cuda, 31 + d)
    per = 320 // page
    tables = _tables(g, 3, per)
    cache = wo.kv4_cache(3 * per + 2, hkv, d, page, device=cuda)
    tok = torch.arange(300, device=cuda)
    for i in range(3):
        ref.write_cache(cache, tables[i], tok, *(_randn(g, 300, hkv, d, dtype=torch.float32) for _ in range(2)))
    starts, lens = [0, 37, 299], [300, 64, 1]
    k_out, v_out = (torch.empty(sum(lens) + 3, hkv, d, dtype=BF, device=cuda).fill_(9.0) for _ in range(2))
    wo.kv4_gather(tables, cache, starts, lens, k_out, v_out, hkv, head_dim=d, page=page)
    at = 0
    for i, (a, n) in enumerate(zip(starts, lens)):
        for (_, x), got in zip(ref.read_cache(cache, tables[i], tok[a:a + n], d), (k_out, v_out)):
            assert torch.equal(got[at:at + n], x.float().to(BF))  # s * code + m is rounded to fp32, then to bf16
        at += n
    assert bool((k_out[at:] == 9.0).all()) and bool((v_out[at:] == 9.0).all())


def _check_cached(dev, rows, ctx, hq, hkv, d, page, seed=0, bias=0.0, scale=None, gain=1.0, bound=0):
    from swarmlora_b200 import worker_ops as wo
    g = _gen(dev, seed)
    n = len(rows)
    longest = max(a + b for a, b in zip(rows, ctx))
    tables = _tables(g, n, -(-longest // page))
    cache = torch.full((tables.numel() + 2, page // 16, hkv, 18 * d), 0xff, dtype=torch.uint8, device=dev)  # NaN pairs
    for i in range(n):
        tok = torch.arange(ctx[i] + rows[i], device=dev)
        ref.write_cache(cache, tables[i], tok, *(_randn(g, tok.numel(), hkv, d, dtype=torch.float32) + bias for _ in range(2)))
    q = _randn(g, sum(rows), hq * d) * gain
    lens = torch.tensor(ctx, dtype=torch.int32, device=dev)
    out = torch.full((sum(rows) + 2, hq * d + 8), 9.0, dtype=BF, device=dev)
    scale = d ** -0.5 if scale is None else scale
    wo.paged_attention_kv4(rows, tables, cache, lens, out, q, hq, hkv, max(longest, bound), scale, head_dim=d, page=page)
    assert bool((out[sum(rows):] == 9.0).all()) and bool((out[:, hq * d:] == 9.0).all())
    at = 0
    for i, r in enumerate(rows):
        tok = torch.arange(ctx[i] + r, device=dev)
        (_, k), (vc, v) = ref.read_cache(cache, tables[i], tok, d)
        # s code and m apart: the parts a value is summed from
        zero = ref.read_cache(_with_codes_zero(cache, d), tables[i], tok, d)[1][1]
        x = q[at:at + r].reshape(r, hq, d)
        _near(out[at:at + r, :hq * d].reshape(r, hq, d), ref.attend_fast(x, k, v, scale),
              ref.attend_fast(x, k, (v - zero).abs() + zero.abs(), scale), f"slot {i} of {rows}/{ctx}")
        at += r


def _with_codes_zero(cache, d):
    c = cache.clone()
    c[..., 9 * d:17 * d] = 0
    return c


@pytest.mark.parametrize("rows,ctx", [
    ([1], [0]), ([1], [14]), ([1], [15]), ([1], [16]), ([1, 1, 1], [255, 256, 700]), ([2], [15]), ([5], [30]), ([16, 1, 0, 3], [100, 0, 9, 333]),
    ([40], [0]), ([1], [5000]), ([3, 1], [2047, 4100])])
@pytest.mark.parametrize("d,hq,hkv,page", [(128, 8, 2, 16), (64, 8, 2, 32), (128, 6, 6, 16), (128, 10, 2, 64), (64, 24, 1, 16)])
def test_cached_attention(native, cuda, rows, ctx, d, hq, hkv, page):
    _check_cached(cuda, rows, ctx, hq, hkv, d, page, seed=sum(ctx) + hq)


def test_cached_attention_of_a_full_decode_step(native, cuda):
    g = torch.Generator().manual_seed(1)
    _check_cached(cuda, [1] * 28, torch.randint(256, 768, (28,), generator=g).tolist(), 32, 8, 128, 16, seed=2)
    _check_cached(cuda, [1] * 128, torch.randint(0, 90, (128,), generator=g).tolist(), 4, 2, 64, 16, seed=3)


@pytest.mark.parametrize("rows,ctx", [
    ([1], [0]), ([1], [40]), ([1, 1, 1], [255, 0, 700]), ([2, 0, 2], [15, 3, 600]), ([4, 1], [1000, 2]), ([16, 1, 0, 3], [100, 0, 9, 333]),
    ([1] * 30, list(range(0, 900, 30)))])
@pytest.mark.parametrize("d,hq,hkv,page", [(128, 8, 2, 16), (64, 8, 2, 32), (128, 6, 6, 16), (64, 24, 1, 16), (128, 32, 8, 16)])
def test_cached_attention_under_a_long_bound(native, cuda, rows, ctx, d, hq, hkv, page):
    """The bound on the contexts is long (the work is cut into equal ranges), the contexts themselves are not."""
    _check_cached(cuda, rows, ctx, hq, hkv, d, page, seed=sum(ctx) + hq + 1, bound=9000)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("hq,hkv,rows,ctx", [
    (32, 8, [1] * 6, [129, 130, 400, 1023, 1500, 3000]), (32, 8, [1] * 36, [600] * 36), (16, 8, [1] * 40, [16 * i for i in range(40)]),
    (64, 8, [1] * 5, [127, 128, 200, 2000, 3100]), (32, 8, [1] * 60, [17 * i for i in range(60)]), (32, 4, [2, 1, 3], [900, 3190, 0])])
def test_cached_attention_by_whole_pairs(native, cuda, d, hq, hkv, rows, ctx):
    _check_cached(cuda, rows, ctx, hq, hkv, d, 16, seed=len(rows) + hq)


def test_cached_attention_offsets_and_large_scores(native, cuda):
    _check_cached(cuda, [1, 4], [333, 1200], 8, 2, 128, 16, seed=4, bias=50.0)
    _check_cached(cuda, [1, 4], [333, 1200], 8, 2, 128, 16, seed=5, gain=20.0)
    _check_cached(cuda, [2], [600], 4, 4, 64, 16, seed=6, scale=3.0)


def test_cached_attention_ignores_what_lies_behind_the_context(native, cuda):
    """Stale tokens of the last page (NaN pairs, any codes) do not reach the rows, and a row
    does not see the tokens appended after it."""
    from swarmlora_b200 import worker_ops as wo
    g = _gen(cuda, 8)
    d, hkv, hq = 128, 2, 8
    tables = torch.arange(4, dtype=torch.int32, device=cuda).reshape(1, 4)
    a = wo.kv4_cache(4, hkv, d, device=cuda)
    ref.write_cache(a, tables[0], torch.arange(40, device=cuda), *(_randn(g, 40, hkv, d, dtype=torch.float32) for _ in range(2)))
    b = a.clone()
    bad = torch.full((24, hkv, d), float("nan"), device=cuda)
    ref.write_cache(b, tables[0], torch.arange(40, 64, device=cuda), bad, bad)
    ref.write_cache(b, tables[0], torch.arange(38, 40, device=cuda), bad[:2], bad[:2])
    q = _randn(g, 3, hq * d)
    lens = torch.tensor([37], dtype=torch.int32, device=cuda)
    outs = [torch.empty(3, hq * d, dtype=BF, device=cuda) for _ in range(2)]
    for c, o in zip((a, b), outs):
        wo.paged_attention_kv4([3], tables, c, lens, o, q, hq, hkv, 64, 0.1)
    assert torch.equal(outs[0][:1], outs[1][:1])
    assert outs[1][1:].isnan().all()


def test_a_prompt_goes_through_all_of_them(native, cuda):
    """A prompt in two chunks and two decoded tokens: append, attention of the first chunk on its own rows,
    gather + attention of the second behind the cached prefix, then the cache's own attention,
    each against 64 bits on what the cache holds; every step captured and replayed once."""
    from swarmlora_b200 import worker_ops as wo
    g = _gen(cuda, 40)
    hq, hkv, d, page, n = 8, 2, 128, 16, 2
    first, second = [50, 33], [21, 64]
    width, scale = (hq + 2 * hkv) * d, d ** -0.5
    cs = _cos_sin(256, d, cuda)
    tables = _tables(g, n, 10)
    cache = wo.kv4_cache(n * 10 + 2, hkv, d, page, device=cuda)
    lens = torch.zeros(n, dtype=torch.int32, device=cuda)

    def append(rows, want_k):
        qkv = _randn(g, sum(rows), width)
        q = torch.empty(sum(rows), hq * d, dtype=BF, device=cuda)
        k = torch.empty(sum(rows), hkv * d, dtype=BF, device=cuda) if want_k else None
        wo.kv4_append(qkv, tables, cache, lens, q, cs, hq, hkv, rows=rows, k_rot=k)
        return qkv, q, k
    qkv, q, k = append(first, True)
    k, v = k.unflatten(-1, (hkv, d)), qkv[:, (hq + hkv) * d:].unflatten(-1, (hkv, d))
    o = wo.prompt_attention(q.unflatten(-1, (hq, d)), k, v, first)
    for a, b, c, got in zip(q.unflatten(-1, (hq, d)).split(first), k.split(first), v.split(first), o.split(first)):
        _near(got, ref.attend_fast(a, b, c, scale), ref.attend_fast(a, b, c.abs(), scale), "first chunk")
    lens += torch.tensor(first, dtype=torch.int32, device=cuda)
    _, q, _ = append(second, False)
    total = [a + b for a, b in zip(first, second)]
    k_all, v_all = (torch.empty(sum(total), hkv, d, dtype=BF, device=cuda) for _ in range(2))
    wo.kv4_gather(tables, cache, [0] * n, total, k_all, v_all, hkv)
    o = wo.prompt_attention(q.unflatten(-1, (hq, d)), k_all, v_all, second, total)
    for a, b, c, got in zip(q.unflatten(-1, (hq, d)).split(second), k_all.split(total), v_all.split(total), o.split(second)):
        _near(got, ref.attend_fast(a, b, c, scale), ref.attend_fast(a, b, c.abs(), scale), "second chunk")
    lens += torch.tensor(second, dtype=torch.int32, device=cuda)
    # decode: append and attention captured once, replayed for two tokens
    qkv = torch.empty(n, width, dtype=BF, device=cuda)
    q, out = (torch.empty(n, hq * d, dtype=BF, device=cuda) for _ in range(2))
    part = torch.empty(max(1, wo.kv4_part_floats([1] * n, hq, hkv, 160)), dtype=torch.float32, device=cuda)

    def step():
        wo.kv4_append(qkv, tables, cache, lens, q, cs, hq, hkv, rows=[1] * n)
        wo.paged_attention_kv4([1] * n, tables, cache, lens, out, q, hq, hkv, 160, scale, part=part)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        step()
    for t in range(2):
        qkv.copy_(_randn(g, n, width))
        graph.replay()
        for i in range(n):
            (_, k), (_, v) = ref.read_cache(cache, tables[i], torch.arange(total[i] + t + 1, device=cuda), d)
            x = q[i].reshape(1, hq, d)
            _near(out[i].reshape(1, hq, d), ref.attend_fast(x, k, v, scale),
                  ref.attend_fast(x, k, v.abs() + 8.0, scale), f"token {t} of slot {i}")
        lens += 1


# ---- strides, streams and far offsets ------------------------------------------------------------
def test_prompt_rows_with_strides(native, cuda):
    """q, k, v and out as row-strided views; what lies between the rows is left alone."""
    from swarmlora_b200 import worker_ops as wo
    g = _gen(cuda, 50)
    lens = [70, 5, 131]
    T, hq, hkv, d = sum(lens), 8, 2, 128

    def view(heads):
        return _randn(g, T, heads * d + 64)[:, 8:8 + heads * d].unflatten(-1, (heads, d))
    q, k, v = view(hq), view(hkv), view(hkv)
    wide = torch.full((T, hq * d + 128), 7.0, dtype=BF, device=cuda)
    out = wide[:, 64:64 + hq * d].unflatten(-1, (hq, d))
    wo.prompt_attention(q, k, v, lens, out=out)
    assert torch.equal(out, wo.prompt_attention(q.contiguous(), k.contiguous(), v.contiguous(), lens))
    assert bool((wide[:, :64] == 7.0).all()) and bool((wide[:, 64 + hq * d:] == 7.0).all())


def test_calls_on_two_streams_at_once(native, cuda):
    """Overlapping calls, each with its own scratch, give what they give alone."""
    from swarmlora_b200 import worker_ops as wo
    g = _gen(cuda, 51)
    hq, hkv, d, n = 8, 2, 128, 3
    tables = _tables(g, n, 130)
    cache = wo.kv4_cache(n * 130 + 2, hkv, d, device=cuda)
    for i in range(n):
        ref.write_cache(cache, tables[i], torch.arange(2000, device=cuda),
                        *(_randn(g, 2000, hkv, d, dtype=torch.float32) for _ in range(2)))
    lens = torch.tensor([1990, 700, 3], dtype=torch.int32, device=cuda)
    qs = [_randn(g, n, hq * d) for _ in range(2)]
    pq, pk, pv = _randn(g, 40, hq, d), _randn(g, 3000, hkv, d), _randn(g, 3000, hkv, d)

    def work(q, out):
        wo.paged_attention_kv4([1] * n, tables, cache, lens, out, q, hq, hkv, 2048, 0.1)
        return wo.prompt_attention(pq, pk, pv, [40], [3000])
    want = []
    for q in qs:
        o = torch.empty(n, hq * d, dtype=BF, device=cuda)
        want.append((o, work(q, o)))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in qs]
    got = [torch.empty(n, hq * d, dtype=BF, device=cuda) for _ in qs]
    prompts = [None, None]
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                prompts[i] = work(qs[i], got[i])
    torch.cuda.synchronize()
    for i in range(2):
        assert torch.equal(got[i], want[i][0]) and torch.equal(prompts[i], want[i][1])


def test_two_graphs_with_their_own_scratch(native, cuda):
    """Attention that needs scratch, captured twice with the scratch left to the call: replays in
    either order and on both streams do not meet."""
    from swarmlora_b200 import worker_ops as wo
    g = _gen(cuda, 52)
    hq, hkv, d = 8, 2, 128
    tables = _tables(g, 1, 300)
    cache = wo.kv4_cache(302, hkv, d, device=cuda)
    ref.write_cache(cache, tables[0], torch.arange(4700, device=cuda),
                    *(_randn(g, 4700, hkv, d, dtype=torch.float32) for _ in range(2)))
    lens = [torch.tensor([n], dtype=torch.int32, device=cuda) for n in (4600, 3100)]
    q = _randn(g, 1, hq * d)
    assert wo.kv4_part_floats([1], hq, hkv, 4800) > 0
    want, outs, graphs, streams = [], [], [], [torch.cuda.Stream(), torch.cuda.Stream()]
    for n, s in zip(lens, streams):
        w, o = (torch.empty(1, hq * d, dtype=BF, device=cuda) for _ in range(2))
        wo.paged_attention_kv4([1], tables, cache, n, w, q, hq, hkv, 4800, 0.1)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            wo.paged_attention_kv4([1], tables, cache, n, o, q, hq, hkv, 4800, 0.1)
        want.append(w)
        outs.append(o)
        graphs.append(graph)
    for _ in range(10):
        for graph, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, outs))


def test_pages_and_rows_beyond_32_bit_offsets(native, cuda):
    """A cache of 5.5 GB whose last pages are used, and prompt rows more than 2^31 elements
    into their tensor."""
    from swarmlora_b200 import worker_ops as wo
    g = _gen(cuda, 53)
    hq, hkv, d, pages = 8, 8, 128, 300_000
    cache = torch.empty(pages, 1, hkv, 18 * d, dtype=torch.uint8, device=cuda)
    small = wo.kv4_cache(4, hkv, d, device=cuda)
    far = torch.tensor([[pages - 1, pages - 3, pages // 2 + 1, 0]], dtype=torch.int32, device=cuda)
    near = torch.tensor([[0, 1, 2, 3]], dtype=torch.int32, device=cuda)
    cache[far[0].long()] = 0
    lens, cs = torch.zeros(1, dtype=torch.int32, device=cuda), _cos_sin(64, d, cuda)
    qkv = _randn(g, 60, (hq + 2 * hkv) * d)
    res = []
    for c, t in ((cache, far), (small, near)):
        q_rot = torch.empty(60, hq * d, dtype=BF, device=cuda)
        k, v = (torch.empty(60, hkv, d, dtype=BF, device=cuda) for _ in range(2))
        out = torch.empty(2, hq * d, dtype=BF, device=cuda)
        wo.kv4_append(qkv, t, c, lens, q_rot, cs, hq, hkv, rows=[60])
        wo.kv4_gather(t, c, [0], [60], k, v, hkv)
        wo.paged_attention_kv4([2], t, c, lens + 58, out, q_rot[:2].contiguous(), hq, hkv, 64, 0.1)
        res.append((q_rot, k, v, out))
    assert all(torch.equal(a, b) for a, b in zip(*res))
    del cache
    rows, stride = 2200, 1 << 20
    big = torch.empty(rows, stride, dtype=BF, device=cuda)
    k, v = (big[:, o:o + 2 * d].unflatten(-1, (2, d)) for o in (0, 4096))
    for t in (k, v):
        t.copy_(_randn(g, rows, 2, d))
    q = _randn(g, 90, 4, d)
    got = wo.prompt_attention(q, k, v, [30, 60], [200, 2000])
    assert torch.equal(got, wo.prompt_attention(q, k.contiguous(), v.contiguous(), [30, 60], [200, 2000]))


def _no_wait_ran_out(native):
    import ctypes as C
    torch.cuda.synchronize()
    code = C.c_uint(7)
    native.check(native.lib().swl_attention_device_error(C.byref(code)))
    return code.value == 0


def test_items_whose_masked_tiles_follow_one_another(native, cuda):
    """Blocks of which only the second row tile reaches the second key tile, mixed with
    blocks of one row tile that crosses into it: four V tiles in a row hold masked keys,
    and the scan of the last may be done while a product still waits for the second."""
    from swarmlora_b200 import worker_ops as wo
    for d, hq, hkv in ((64, 64, 8), (128, 64, 8), (64, 8, 8)):
        two, one = (32, 136), (16, 136)  # tokens, keys at a group of 8
        lens = [two, one, one] * 20 if hq > hkv else [(256, 264), (128, 264)] * 20
        q_lens, k_lens = [a for a, _ in lens], [b for _, b in lens]
        first = _check_prompt(cuda, q_lens, k_lens, hq, hkv, d, seed=11)
        g = _gen(cuda, 11)
        q, k, v = (_randn(g, sum(n), h, d) for n, h in ((q_lens, hq), (k_lens, hkv), (k_lens, hkv)))
        for _ in range(100):
            again = wo.prompt_attention(q, k, v, q_lens, k_lens, scale=d ** -0.5)
        assert torch.equal(again, first) and _no_wait_ran_out(native)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("group", [1, 2, 5, 8])
def test_mixed_batches_are_the_same_every_time(native, cuda, d, group):
    from swarmlora_b200 import worker_ops as wo
    import random
    r = random.Random(d + group)
    for n in (3, 14, 40):
        q_lens = [r.choice([1, 7, 16, 33, 100, 128, 130, 266, 500]) for _ in range(n)]
        k_lens = [a + r.choice([0, 0, 3, 10, 120, 700]) for a in q_lens]
        hkv = 8 // group if group < 8 else 4
        g = _gen(cuda, n)
        q, k, v = (_randn(g, sum(m), h, d) for m, h in ((q_lens, hkv * group), (k_lens, hkv), (k_lens, hkv)))
        first = wo.prompt_attention(q, k, v, q_lens, k_lens)
        outs = [wo.prompt_attention(q, k, v, q_lens, k_lens) for _ in range(30)]
        assert all(torch.equal(o, first) for o in outs)
    assert _no_wait_ran_out(native)


def test_no_wait_ran_out(native, cuda):
    """The bounded-wait status after this file's launches (it is cleared by reading)."""
    import ctypes as C
    torch.cuda.synchronize()
    code = C.c_uint(7)
    native.check(native.lib().swl_attention_device_error(C.byref(code)))
    assert code.value == 0
