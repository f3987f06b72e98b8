"""What the 4-bit cache calls take and refuse, without a GPU: the slots' own tables and
caches, and what the host side makes of them."""
import ctypes as C

import pytest
import torch

F = 0x1000  # an aligned address that is never dereferenced


def _each(native, call, rows=(1, 1), table_lens=(4, 2), pages=(8, 3), starts=(0, 0), null=()):
    n, lib, p = len(rows), native.lib(), native.ptr_array
    ptrs = p([F] * n)
    lens = None if "table_lens" in null else native.i32_array(table_lens)
    count = None if "pages" in null else (C.c_int64 * n)(*pages)
    counts = native.i32_array(rows)
    if call == "append":
        st = lib.swl_kv4_append_each(n, counts, ptrs, 1024, ptrs, lens, ptrs, count, ptrs, 4, 2, 128, 16, F, 64, F, None, None)
    elif call == "gather":
        st = lib.swl_kv4_gather_each(n, native.i32_array(starts), counts, ptrs, lens, ptrs, count, 2, 128, 16, F, F, None)
    else:
        st = lib.swl_paged_attention_kv4_each(n, counts, ptrs, lens, ptrs, count, ptrs, ptrs, 512, 4, 2, 128, 16, 0.1, 64, F,
                                              None, None)
    return st, native.last_error()


@pytest.mark.parametrize("call", ["append", "gather", "attention"])
@pytest.mark.parametrize("bad,word", [
    (dict(null=("table_lens",)), "null table lengths"), (dict(null=("pages",)), "page counts"),
    (dict(table_lens=(4, 0)), "empty"), (dict(pages=(0, 3)), "empty"), (dict(pages=(8, -1)), "empty")])
def test_slots_of_their_own_sizes_refuse(native, call, bad, word):
    st, msg = _each(native, call, **bad)
    assert st != 0 and word in msg, (st, msg)


def test_a_gather_is_bounded_by_the_slots_own_table(native):
    st, msg = _each(native, "gather", rows=(64, 33))
    assert st != 0 and "33 of slot 1 lie outside" in msg, msg


def test_each_slot_keeps_its_own_sizes(native):
    from swarmlora_b200 import worker_ops as wo
    pages = [8, 3, 5]
    caches = [wo.kv4_cache(n, 2, device="cpu") for n in pages]
    tables = [torch.zeros(n, dtype=torch.int32) for n in (2, 6, 1)]
    _, lens, _, count = wo._kv4_slots(tables, caches, 3, 2, 128, 16, -1)
    assert list(lens) == [2, 6, 1] and list(count) == pages
    # one row of a table of tables is as good as the row itself
    _, lens, _, _ = wo._kv4_slots([torch.zeros(4, 7, dtype=torch.int32)[i:i + 1] for i in range(3)], caches, 3, 2, 128, 16, -1)
    assert list(lens) == [7, 7, 7]
    _, lens, _, count = wo._kv4_slots(torch.zeros(3, 5, dtype=torch.int32), caches[0], 3, 2, 128, 16, -1)
    assert list(lens) == [5, 5, 5] and list(count) == [8, 8, 8]
    for bad in (torch.zeros(2, 7, dtype=torch.int32), torch.tensor(1, dtype=torch.int32)):
        with pytest.raises(ValueError, match="block tables"):
            wo._kv4_slots([bad] * 3, caches, 3, 2, 128, 16, -1)


def test_packed_rows_are_contiguous_inside(native):
    """Packed rows beside listed tables: rows whose elements lie apart are refused."""
    from swarmlora_b200 import worker_ops as wo
    rows = torch.zeros(3, 8, dtype=torch.bfloat16)
    first = [0, 2]
    got = wo._slot_rows(rows[:, :6], 2, "rows", torch.bfloat16, 2, -1, first)
    assert list(got) == [rows.data_ptr(), rows.data_ptr() + 2 * 16]
    for bad in (torch.zeros(8, 3, dtype=torch.bfloat16).t(), torch.zeros(3, 16, dtype=torch.bfloat16)[:, ::2], rows.float()):
        with pytest.raises(ValueError, match="rows"):
            wo._slot_rows(bad, 2, "rows", torch.bfloat16, 2, -1, first)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("rows", [[1], [1] * 28, [5] * 28])
def test_the_largest_bound_plans_as_a_long_one_does(native, d, rows):
    from swarmlora_b200 import worker_ops as wo
    long = wo.kv4_part_floats(rows, 32, 8, 1 << 20, head_dim=d)
    assert long > 0
    for bound in (2 ** 31 - 17, 2 ** 31 - 16, 2 ** 31 - 15, 2 ** 31 - 1):
        assert wo.kv4_part_floats(rows, 32, 8, bound, head_dim=d) == long, bound


@pytest.mark.parametrize("rows", [(), (0,), (0, 0, 0)])
def test_calls_without_a_row_need_no_tensors(native, rows):
    """Empty tensors have no address."""
    n, lib = len(rows), native.lib()
    counts, none, zeros = native.i32_array(rows or (0,)), native.ptr_array([None] * max(n, 1)), native.i32_array([0] * max(n, 1))
    pages = (C.c_int64 * max(n, 1))(*[0] * max(n, 1))
    calls = [
        lib.swl_kv4_append(n, counts, none, 1024, none, 0, none, 0, none, 4, 2, 128, 16, F, 64, None, None, None),
        lib.swl_kv4_append_each(n, counts, none, 1024, none, zeros, none, pages, none, 4, 2, 128, 16, F, 64, None, None, None),
        lib.swl_kv4_append_packed(n, counts, None, 1024, None, 0, 0, None, 0, None, 4, 2, 128, 16, F, 64, None, None, None),
        lib.swl_kv4_gather(n, zeros, counts, none, 0, none, 0, 2, 128, 16, None, None, None),
        lib.swl_kv4_gather_each(n, zeros, counts, none, zeros, none, pages, 2, 128, 16, None, None, None),
        lib.swl_kv4_gather_packed(n, zeros, counts, None, 0, 0, None, 0, 2, 128, 16, None, None, None),
        lib.swl_paged_attention_kv4(n, counts, none, 0, none, 0, none, none, 512, 4, 2, 128, 16, 0.1, 64, None, None, None),
        lib.swl_paged_attention_kv4_each(n, counts, none, zeros, none, pages, none, none, 512, 4, 2, 128, 16, 0.1, 64, None,
                                         None, None),
        lib.swl_paged_attention_kv4_packed(n, counts, None, 0, 0, None, 0, None, None, 512, 4, 2, 128, 16, 0.1, 64, None, None,
                                           None)]
    assert calls == [0] * len(calls), native.last_error()


def test_a_stream_of_another_device_is_refused(native):
    from types import SimpleNamespace
    from swarmlora_b200 import worker_ops as wo
    assert wo._elsewhere(0, SimpleNamespace(device_index=1))
    with pytest.raises(ValueError, match="stream belongs to cuda:1"):
        wo._there(0, SimpleNamespace(device_index=1))


def test_a_wait_that_ran_out_is_reported(native, monkeypatch):
    """The error word and a failing read reach the caller (the library's part is a stand-in)."""
    import contextlib
    from swarmlora_b200 import worker_ops as wo
    seen, status = [], [0]

    class Lib:
        def swl_attention_device_error(self, code):
            code._obj.value = 111
            return status[0]
    monkeypatch.setattr(wo, "lib", Lib)
    monkeypatch.setattr(torch.cuda, "device", lambda d: (seen.append(d), contextlib.nullcontext())[1])
    assert wo.attention_device_error() == 111 and wo.attention_device_error(3) == 111 and seen == [None, 3]
    status[0] = 2
    with pytest.raises(RuntimeError):
        wo.attention_device_error()


def test_the_stride_of_a_single_entry_does_not_count(native):
    """One slot's length as a column of a wider table, one page a table as a transposed row."""
    from swarmlora_b200 import worker_ops as wo
    meta = torch.zeros(4, 6, dtype=torch.int32)
    assert wo._check_slots("seqlens", meta[1:2, 3], 1, torch.int32, -1, 1) == 6
    assert wo._check_slots("block tables", meta[:1].t()[2:5], 3, torch.int32, -1, 2) == 1
    assert list(wo._slot_rows(meta[1:2, 3], 1, "seqlens", torch.int32, 4, -1)) == [meta[1, 3].data_ptr()]
    for bad, n, dims in ((meta[:, 3], 4, 1), (meta.t(), 6, 2)):
        with pytest.raises(ValueError, match="contiguous inside"):
            wo._check_slots("tables", bad, n, torch.int32, -1, dims)


def test_torch_without_the_shortcuts(native, monkeypatch):
    """The current stream and device come from torch's public calls where the private ones are missing."""
    import importlib.util
    from types import SimpleNamespace
    from swarmlora_b200 import worker_ops as wo
    for name in ("_cuda_getCurrentRawStream", "_cuda_getDevice"):
        monkeypatch.delattr(torch._C, name, raising=False)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda at: SimpleNamespace(cuda_stream=100 + at))
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 2)
    spec = importlib.util.spec_from_file_location("swarmlora_b200.worker_ops_plain", wo.__file__)
    plain = importlib.util.module_from_spec(spec)
    monkeypatch.setitem(__import__("sys").modules, spec.name, plain)  # (dataclasses look their module up)
    spec.loader.exec_module(plain)
    assert plain._current(3) == 103 and plain._elsewhere(1, None) and not plain._elsewhere(2, None)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("rows,hq,hkv,whole", [
    ([1] * 28, 32, 8, 2816), ([1], 40, 8, 2816), ([2, 1], 32, 8, 2816),    # one column tile, pairs that fit at a time
    ([1] * 60, 32, 8, 2176),                                                # more pairs than fit
    ([2, 1, 3], 32, 4, 5120), ([4, 1], 32, 8, 5120),                        # two column tiles
    ([5] * 28, 32, 8, 2176)])                                               # and more pairs than fit
def test_up_to_which_bound_whole_pairs_are_taken(native, d, rows, hq, hkv, whole):
    """(Where no device says how many multiprocessors it has, the plan counts 148.)"""
    from swarmlora_b200 import worker_ops as wo
    assert wo.kv4_part_floats(rows, hq, hkv, whole, head_dim=d) == 0
    assert wo.kv4_part_floats(rows, hq, hkv, whole + 1, head_dim=d) > 0
