"""Refusals of the prompt and 4-bit cache entry points (no GPU: every call fails before
any device work), the cache's block size, and the plain forms that the GPU
tests compare with."""
import ctypes as C

import pytest
import torch

from tests import kv4_reference as ref

F = 0x1000  # an aligned address that is never dereferenced


def _prompt(native, q_lens=(4,), k_lens=(4,), q=F, qs=512, k=F, ks=256, v=F, vs=256, out=F, os=512, hq=4, hkv=2, d=128,
            scale=0.1, n=None):
    st = native.lib().swl_prompt_attention(len(q_lens) if n is None else n, native.i32_array(q_lens),
                                           native.i32_array(k_lens), q, qs, k, ks, v, vs, out, os, hq, hkv, d, scale,
                                           None, None)
    return st, native.last_error()


@pytest.mark.parametrize("bad,word", [
    (dict(d=96), "head_dim"), (dict(hq=5), "multiple"), (dict(hkv=0), "multiple"), (dict(scale=0.0), "scale"),
    (dict(scale=-1.0), "scale"), (dict(scale=float("nan")), "scale"), (dict(scale=float("inf")), "scale"),
    (dict(qs=504), "strides"), (dict(ks=248), "strides"), (dict(qs=516), "multiples of 8"), (dict(vs=260), "multiples of 8"),
    (dict(q=None), "null"), (dict(k=None), "null"), (dict(out=None), "null"), (dict(v=F + 8), "aligned"),
    (dict(q_lens=(-1,)), "negative"), (dict(n=129, q_lens=(1,) * 129, k_lens=(1,) * 129), "segment count"),
    (dict(q_lens=(1 << 30, 1), k_lens=(1, 1)), "2^30"),
    (dict(hq=258, hkv=2, qs=1 << 16, os=1 << 16), "at most 128"),
])
def test_prompt_attention_refuses(native, bad, word):
    st, msg = _prompt(native, **bad)
    assert st != 0 and word in msg, (st, msg)


def test_prompt_attention_of_nothing_is_done(native):
    assert _prompt(native, q_lens=(0, 0), k_lens=(0, 3))[0] == 0
    assert _prompt(native, q_lens=(), k_lens=(), n=0)[0] == 0


def _kv4(native, call, rows=(1,), hq=4, hkv=2, d=128, page=16, table_len=4, pages=8, bt=F, cache=F, seqlen=F, qkv=F,
         stride=None, cs=F, max_pos=64, q_rot=F, k_rot=None, starts=(0,), k_out=F, v_out=F, out=F, out_stride=None,
         scale=0.1, max_len=64):
    n = len(rows)
    lib, p = native.lib(), native.ptr_array
    tables, caches, lens = p([bt] * n), p([cache] * n), p([seqlen] * n)
    if call == "append":
        st = lib.swl_kv4_append(n, native.i32_array(rows), p([qkv] * n), stride or (hq + 2 * hkv) * d, tables, table_len,
                                caches, pages, lens, hq, hkv, d, page, cs, max_pos, q_rot, k_rot, None)
    elif call == "gather":
        st = lib.swl_kv4_gather(n, native.i32_array(starts), native.i32_array(rows), tables, table_len, caches, pages, hkv,
                                d, page, k_out, v_out, None)
    else:
        st = lib.swl_paged_attention_kv4(n, native.i32_array(rows), tables, table_len, caches, pages, lens, p([out] * n),
                                         out_stride or hq * d, hq, hkv, d, page, scale, max_len, q_rot, None, None)
    return st, native.last_error()


@pytest.mark.parametrize("call", ["append", "gather", "attention"])
@pytest.mark.parametrize("bad,word", [
    (dict(d=32), "head_dim"), (dict(hkv=0), "kv heads"), (dict(page=8), "page"), (dict(page=48), "page"),
    (dict(page=2048), "page"), (dict(table_len=0), "empty"), (dict(pages=0), "empty"), (dict(bt=None), "null"),
    (dict(cache=None), "null"), (dict(cache=F + 8), "aligned"), (dict(rows=(-1,)), "negative"),
    (dict(rows=(0,) * 129, starts=(0,) * 129), "segment count"),
])
def test_kv4_calls_refuse(native, call, bad, word):
    st, msg = _kv4(native, call, **bad)
    assert st != 0 and word in msg, (st, msg)


@pytest.mark.parametrize("call,bad,word", [
    ("append", dict(hq=0), "query heads"), ("append", dict(max_pos=0), "cos/sin"), ("append", dict(cs=None), "cos/sin"),
    ("append", dict(q_rot=None), "q_rot"), ("append", dict(stride=1016), "stride"), ("append", dict(stride=1028), "stride"),
    ("append", dict(qkv=None), "null"), ("append", dict(qkv=F + 2), "aligned"), ("append", dict(k_rot=F + 4), "aligned"),
    ("append", dict(seqlen=None), "null"), ("gather", dict(starts=(-1,)), "outside"),
    ("gather", dict(starts=(60,), rows=(5,)), "outside"), ("gather", dict(k_out=None), "aligned"),
    ("gather", dict(v_out=F + 8), "aligned"), ("attention", dict(hq=5), "multiple"), ("attention", dict(scale=0.0), "scale"),
    ("attention", dict(max_len=0), "max_len"), ("attention", dict(q_rot=None), "aligned"),
    ("attention", dict(out_stride=508), "stride"), ("attention", dict(out=None), "aligned"),
    ("attention", dict(seqlen=None), "null"),
])
def test_kv4_call_refuses_its_own(native, call, bad, word):
    st, msg = _kv4(native, call, **bad)
    assert st != 0 and word in msg, (st, msg)


@pytest.mark.parametrize("bad,word", [
    (dict(d=96), "head_dim"), (dict(page=24), "page"), (dict(bt=None), "null"), (dict(cache=None), "null"),
    (dict(cache=F + 8), "aligned"), (dict(rows=(-1,)), "negative"), (dict(table_len=0), "empty"), (dict(pages=0), "empty"),
    (dict(rows=(1,) * 129), "segment count"), (dict(seqlen=None), "null")])
def test_packed_kv4_calls_refuse(native, bad, word):
    a = dict(rows=(1,), d=128, page=16, table_len=4, pages=8, bt=F, cache=F, seqlen=F) | bad
    lib, n, rows = native.lib(), len(a["rows"]), native.i32_array(a["rows"])
    calls = [lib.swl_kv4_append_packed(n, rows, F, 1024, a["bt"], 4, a["table_len"], a["cache"], a["pages"], a["seqlen"], 4, 2,
                                       a["d"], a["page"], F, 64, F, None, None), native.last_error(),
             lib.swl_paged_attention_kv4_packed(n, rows, a["bt"], 4, a["table_len"], a["cache"], a["pages"], a["seqlen"], F, 512,
                                                4, 2, a["d"], a["page"], 0.1, 64, F, None, None), native.last_error()]
    if "seqlen" not in bad:
        calls += [lib.swl_kv4_gather_packed(n, native.i32_array([0] * n), rows, a["bt"], 4, a["table_len"], a["cache"],
                                            a["pages"], 2, a["d"], a["page"], F, F, None), native.last_error()]
    for st, msg in zip(calls[::2], calls[1::2]):
        assert st != 0 and word in msg, (st, msg)


def test_error_word_needs_a_place(native):
    assert native.lib().swl_attention_device_error(None) != 0 and "null" in native.last_error()


@pytest.mark.parametrize("call", ["append", "gather", "attention"])
def test_kv4_calls_of_nothing_are_done(native, call):
    assert _kv4(native, call, rows=(0, 0), starts=(0, 64))[0] == 0


def test_block_bytes(native):
    from swarmlora_b200 import worker_ops as wo
    assert [native.lib().swl_kv4_block_bytes(d) for d in (64, 128, 96)] == [1152, 2304, 0]
    assert [wo.kv4_block_bytes(d) for d in (64, 128)] == [1152, 2304]


def test_python_entry_points_refuse_host_tensors(native):
    from swarmlora_b200 import worker_ops as wo
    q = torch.zeros(2, 4, 128, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="CUDA"):
        wo.prompt_attention(q, q, q, [2])
    with pytest.raises(ValueError, match="CUDA"):
        wo.kv4_append(q.flatten(1), [], [], [], q.flatten(1), q[0], 2, 1, rows=[2])
    with pytest.raises(ValueError, match="CUDA"):
        wo.kv4_gather([], [], [0], [1], q, q, 4)
    with pytest.raises(ValueError, match="CUDA"):
        wo.paged_attention_kv4([1], [], [], [], q.flatten(1), q.flatten(1), 4, 2, 16, 0.1)
    with pytest.raises(ValueError, match="head_dim"):
        wo.kv4_cache(2, 2, head_dim=96, device="cpu")
    with pytest.raises(ValueError, match="page"):
        wo.kv4_cache(2, 2, page=24, device="cpu")


@pytest.mark.parametrize("d", [64, 128])
def test_layout_covers_every_bit_once(d):
    """The codes and pairs of a block's 16 tokens fill its 18 D bytes exactly."""
    seen = torch.zeros(18 * d, 2, dtype=torch.long)
    for t in range(16):
        for i in range(d):
            for at, shift, _ in ref.offsets(d, t, i):
                seen[at, shift // 4] += 1
        for i in range(0, d, 64):
            for _, _, pair in ref.offsets(d, t, i):
                seen[pair:pair + 4] += 1
    assert bool((seen == 1).all())


def test_written_cache_reads_back():
    g = torch.Generator().manual_seed(1)
    d, hkv, page = 128, 3, 32
    cache = torch.zeros(4, page // 16, hkv, 18 * d, dtype=torch.uint8)
    table = torch.tensor([2, 0, 3], dtype=torch.int32)
    tok = torch.tensor([0, 5, 31, 32, 70, 95])
    k, v = torch.randn(6, hkv, d, generator=g), 3 + torch.randn(6, hkv, d, generator=g)
    ref.write_cache(cache, table, tok, k, v)
    for (code, got), x in zip(ref.read_cache(cache, table, tok, d), (k, v)):
        c, s, m = ref.quantise(x)
        assert torch.equal(code, c) and torch.equal(got, ref.values(c, s, m))
        # half a step, and what rounding s and m to bf16 (2^-8 at most) moves the ends by
        step = s.double().expand(-1, -1, -1, 64).flatten(-2)
        slack = 2.0 ** -8 * (15 * step + m.double().abs().expand(-1, -1, -1, 64).flatten(-2))
        assert bool(((got - x.double()).abs() <= step / 2 + slack).all())
