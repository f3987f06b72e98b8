"""Worker-side kernels (LoRA delta, RoPE + paged KV append, paged attention,
RMSNorm) over one or many slots, through libswarmlora_b200.so.

A worker process normally calls these for its single slot; the benchmark
calls them for all slots at once. Adapter weights are packed once into the
layouts the kernels read (`pack_lora_layer`), following the reference's
FusedLoRA packing (model_builder.py:217-262): the fused QKV / Gate+Up A
matrices are pre-scaled by alpha/r in bf16, O / Down scale after the expand
(worker_sync.py:305, :375).
"""
from __future__ import annotations

import contextlib
import ctypes as C
import itertools
from array import array
from dataclasses import dataclass

import torch

from ._native import check, i32_array, lib, ptr_array

EXPAND_ADD, EXPAND_RESIDUAL, EXPAND_SILU_MUL = 0, 1, 2


def _stream(stream):
    return (stream if stream is not None else torch.cuda.current_stream()).cuda_stream


def _ptrs(ts):
    return ptr_array([t.data_ptr() if t is not None else None for t in ts])


@dataclass
class LoraLayer:
    """One layer of one adapter, in kernel layout (all bf16, on device)."""
    A_qkv: torch.Tensor   # [H, 3r]  = cat(Aq^T s, Ak^T s, Av^T s)
    B_qkv: torch.Tensor   # [q+k+v, r] = cat(Bq, Bk, Bv)
    A_o: torch.Tensor     # [H, r]   = Ao^T
    B_o: torch.Tensor     # [H, r]
    A_gu: torch.Tensor    # [H, 2r]  = cat(Ag^T s, Au^T s)
    B_gu: torch.Tensor    # [2I, r]  = cat(Bg, Bu)
    A_down: torch.Tensor  # [I, r]   = Ad^T
    B_down: torch.Tensor  # [H, r]
    rank: int
    scaling: float


def pack_lora_layer(w: dict, scaling: float, pad_rank: int | None = None,
                    post_scale: float | None = None) -> LoraLayer:
    """w maps 'q','k','v','o','gate','up','down' -> (lora_A [r, in], lora_B [out, r]).

    pad_rank packs the adapter at a larger rank (a group whose adapters have
    different ranks runs its kernels at the largest): A and B get zero
    columns, which add exact zeros, so the deltas are bit-identical.
    post_scale is the scale the O / Down kernels apply after the expand (one
    value per launch); the adapter's own `scaling` is reached by folding
    scaling / post_scale into its O and Down lora_B, which is exact when that
    ratio is a power of two (alpha / r for r in {8, 16, 32} and one alpha)."""
    r = int(w["q"][0].shape[0])
    R = int(pad_rank) if pad_rank else r
    if R < r:
        raise ValueError(f"pad_rank {R} below the adapter's rank {r}")
    fold = 1.0 if post_scale is None else float(scaling) / float(post_scale)

    def pad(t):  # [rows, r] -> [rows, R]
        return torch.nn.functional.pad(t, (0, R - t.shape[1])) if R > t.shape[1] else t

    def a_scaled(name):
        return pad((w[name][0].t() * scaling).to(torch.bfloat16))  # A.t() * s in bf16 (model_builder.py:237)

    def b_folded(name):
        b = w[name][1]
        return pad((b.float() * fold).to(torch.bfloat16) if fold != 1.0 else b)

    return LoraLayer(
        A_qkv=torch.cat([a_scaled("q"), a_scaled("k"), a_scaled("v")], 1).contiguous(),
        B_qkv=torch.cat([pad(w["q"][1]), pad(w["k"][1]), pad(w["v"][1])], 0).contiguous(),
        A_o=pad(w["o"][0].t()).contiguous(),
        B_o=b_folded("o").contiguous(),
        A_gu=torch.cat([a_scaled("gate"), a_scaled("up")], 1).contiguous(),
        B_gu=torch.cat([pad(w["gate"][1]), pad(w["up"][1])], 0).contiguous(),
        A_down=pad(w["down"][0].t()).contiguous(),
        B_down=b_folded("down").contiguous(),
        rank=R,
        scaling=float(post_scale) if post_scale is not None else float(scaling),
    )


LORA_FIELDS = ("A_qkv", "B_qkv", "A_o", "B_o", "A_gu", "B_gu", "A_down", "B_down")
_SLAB_ALIGN = 256  # elements: every tensor of a slab starts on a 512-byte boundary, as torch allocates


@dataclass
class PackedAdapter:
    """All layers of one adapter in one contiguous bf16 buffer (`slab`);
    `layers` are LoraLayers whose tensors are views into it. Adapters packed
    at the same rank for the same model share the layout, so a slot's adapter
    is replaced by one device copy of the slab."""
    slab: torch.Tensor
    layers: list
    rank: int            # the adapter's own rank (the slab holds it padded)


def pack_lora_slab(layers: list, rank: int | None = None) -> PackedAdapter:
    """Copies packed layers (pack_lora_layer) into one slab, fields in
    LORA_FIELDS order layer after layer."""
    offs, total = [], 0
    for L in layers:
        row = []
        for f in LORA_FIELDS:
            t = getattr(L, f)
            row.append((total, tuple(t.shape)))
            total += -(-t.numel() // _SLAB_ALIGN) * _SLAB_ALIGN
        offs.append(row)
    slab = torch.empty(total, dtype=torch.bfloat16, device=layers[0].A_qkv.device)
    views = []
    for L, row in zip(layers, offs):
        kw = {}
        for f, (o, shape) in zip(LORA_FIELDS, row):
            n = shape[0] * shape[1]
            v = slab[o:o + n].view(shape)
            v.copy_(getattr(L, f))
            kw[f] = v
        views.append(LoraLayer(**kw, rank=L.rank, scaling=L.scaling))
    return PackedAdapter(slab, views, int(rank) if rank is not None else layers[0].rank)


def lora_shrink(xs, As, K: int, R: int, splits: int, ws: torch.Tensor, x_stride: int | None = None,
                rows=None, stream=None) -> None:
    rows = rows if rows is not None else [int(x.shape[0]) for x in xs]
    x_stride = x_stride if x_stride is not None else int(xs[0].stride(0))
    check(lib().swl_lora_shrink(len(xs), i32_array(rows), _ptrs(xs), x_stride, _ptrs(As), K, R,
                                splits, ws.data_ptr(), _stream(stream)))


def lora_expand(bases, Bs, outs, n_total: int, r: int, block_ends, mode: int, splits: int,
                ws: torch.Tensor, resids=None, post_scale: float = 0.0, rows=None,
                base_stride: int | None = None, out_stride: int | None = None,
                resid_stride: int = 0, stream=None) -> None:
    rows = rows if rows is not None else [int(b.shape[0]) for b in bases]
    base_stride = base_stride if base_stride is not None else int(bases[0].stride(0))
    out_stride = out_stride if out_stride is not None else int(outs[0].stride(0))
    be = (C.c_int64 * 3)(*[int(x) for x in block_ends] + [n_total] * (3 - len(block_ends)))
    check(lib().swl_lora_expand(
        len(bases), i32_array(rows), _ptrs(bases), base_stride,
        _ptrs(Bs) if Bs is not None else None,
        _ptrs(resids) if resids is not None else None, resid_stride,
        _ptrs(outs), out_stride, n_total, r, len(block_ends), be, float(post_scale), mode, splits,
        ws.data_ptr(), _stream(stream)))


def rope_append(qkvs, block_tables, k_caches, v_caches, seqlens, q_rot, cos_sin, hq: int, hkv: int,
                head_dim: int = 128, page: int = 16, rows=None, qkv_stride: int | None = None,
                stream=None) -> None:
    rows = rows if rows is not None else [int(q.shape[0]) for q in qkvs]
    qkv_stride = qkv_stride if qkv_stride is not None else int(qkvs[0].stride(0))
    check(lib().swl_rope_append(len(qkvs), i32_array(rows), _ptrs(qkvs), qkv_stride,
                                _ptrs(block_tables), _ptrs(k_caches), _ptrs(v_caches),
                                _ptrs(seqlens), hq, hkv, head_dim, page, cos_sin.data_ptr(),
                                int(cos_sin.shape[0]), q_rot.data_ptr(), _stream(stream)))


def attention_tune(chunk_pages: int = 0, stages: int = 0, groups: int = 0) -> None:
    """Pages per context chunk, page-ring depth and kv head groups (CTAs that
    share one page's heads) of the attention launch (0 = automatic)."""
    check(lib().swl_attention_tune(chunk_pages, stages, groups))


def attention_tma(on: bool = True) -> None:
    """K/V pages by TMA (default, when every row's pages share one cache
    allocation) or by per-lane copies."""
    check(lib().swl_attention_tma(1 if on else 0))


def attention_part_floats(total_rows: int, hq: int, hkv: int, max_len: int) -> int:
    return int(lib().swl_attention_part_floats(total_rows, hq, hkv, max_len))


def paged_attention(rows, block_tables, k_caches, v_caches, seqlens, outs, q_rot, part, hq: int,
                    hkv: int, max_len: int, scale: float, head_dim: int = 128, page: int = 16,
                    out_stride: int | None = None, stream=None) -> None:
    out_stride = out_stride if out_stride is not None else int(outs[0].stride(0))
    check(lib().swl_paged_attention(len(rows), i32_array(rows), _ptrs(block_tables),
                                    _ptrs(k_caches), _ptrs(v_caches), _ptrs(seqlens), _ptrs(outs),
                                    out_stride, hq, hkv, head_dim, page, float(scale), max_len,
                                    q_rot.data_ptr(), part.data_ptr() if part is not None else None,
                                    _stream(stream)))


def paged_attention_noalloc(rows, block_tables, k_caches, v_caches, seqlens, outs, q_rot, hq: int,
                            hkv: int, max_len: int, scale: float, head_dim: int = 128,
                            page: int = 16, out_stride: int | None = None, stream=None) -> None:
    """paged_attention with its partials in the library's static per-device
    array (NOALLOC_ATTN_SCRATCH_FLOATS fp32): allocates nothing. Calls that
    overlap on the GPU share that array and must not run concurrently."""
    out_stride = out_stride if out_stride is not None else int(outs[0].stride(0))
    check(lib().swl_paged_attention_noalloc(len(rows), i32_array(rows), _ptrs(block_tables),
                                            _ptrs(k_caches), _ptrs(v_caches), _ptrs(seqlens),
                                            _ptrs(outs), out_stride, hq, hkv, head_dim, page,
                                            float(scale), max_len, q_rot.data_ptr(),
                                            _stream(stream)))


NOALLOC_ATTN_SCRATCH_FLOATS = 1 << 20


# ---- whole prompts, and the key/value cache held in 4 bits --------------------------------------
# A decode step makes these calls once a layer with kernels of a few microseconds, so their
# host side is kept short: tables go through array.array, contexts are entered only where
# needed, and devices are compared by number (`at`: the CUDA device of the call).
_BF16 = torch.bfloat16


def _elsewhere(at: int, stream) -> bool:
    """Whether a call has to switch to its tensors' device or to a stream of its own."""
    return at < 0 or stream is not None or at != _device()


# The current stream's handle and the current device, without making objects of them (3 us); torch's
# public calls where it has no such shortcuts.
_current = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda at: torch.cuda.current_stream(at).cuda_stream)
_device = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device


def _there(at: int, stream):
    if at < 0:
        raise ValueError("CUDA tensors are needed")
    if stream is not None and stream.device_index != at:  # entering it would make its device the current one
        raise ValueError(f"the stream belongs to cuda:{stream.device_index}, the tensors to cuda:{at}")
    ctx = contextlib.ExitStack()
    ctx.enter_context(torch.cuda.device(at))
    ctx.enter_context(torch.cuda.stream(stream))
    return ctx


def _ints(values) -> array:
    return array("i", values)


def _addr(table: array) -> int:
    return table.buffer_info()[0]


def _bf16_rows(name: str, t: torch.Tensor, at: int, heads=None, head_dim=None) -> tuple:
    """A bf16 tensor [rows, heads, head_dim] on the call's device whose heads are
    contiguous: its rows, heads, head_dim and the elements between rows."""
    if t.dtype is not _BF16 or t.get_device() != at:
        raise ValueError(f"{name}: a bf16 tensor on the call's CUDA device is needed")
    shape = t.shape
    if len(shape) != 3 or (heads is not None and shape[1] != heads) or (head_dim is not None and shape[2] != head_dim):
        raise ValueError(f"{name}: shape {tuple(shape)} does not fit")
    n, h, d = shape
    by, st, one = t.stride()
    if one != 1 or (h > 1 and st != d):
        if t.numel():
            raise ValueError(f"{name}: heads must be contiguous")
    return n, h, d, by if n > 1 else -(-h * d // 8) * 8  # a single row's stride is never used (torch leaves it arbitrary)


def _row_stride(t: torch.Tensor) -> int:
    """Elements between rows of a [rows, width] tensor; a single row's stride is never used."""
    n, width = t.shape
    return t.stride()[0] if n > 1 else -(-width // 8) * 8


def prompt_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, q_lens, k_lens=None, scale: float | None = None,
                     out: torch.Tensor | None = None, stream=None) -> torch.Tensor:
    """Causal GQA attention of packed sequences: q [sum q_lens, hq, D], k and v
    [sum k_lens, hkv, D] (row-strided views allowed), lengths on the host. Row
    r of a sequence sees its keys 0 .. r + k_len - q_len (k_lens defaults to
    q_lens; longer ones hold a prefix); a row without keys gives zeros.
    Returns out [rows of q, hq, D] (rows behind the last sequence are left as they are)."""
    at = q.get_device()
    if _elsewhere(at, stream):
        with _there(at, stream):
            return prompt_attention(q, k, v, q_lens, k_lens, scale, out)
    q_rows, hq, D, q_by = _bf16_rows("q", q, at)
    k_rows, hkv, _, k_by = _bf16_rows("k", k, at, None, D)
    v_rows, _, _, v_by = _bf16_rows("v", v, at, hkv, D)
    if k_lens is None:
        k_lens = q_lens
    n, total = len(q_lens), sum(q_lens)
    if len(k_lens) != n:
        raise ValueError("prompt_attention: one key length per sequence")
    if total > q_rows or sum(k_lens) > min(k_rows, v_rows):
        raise ValueError("prompt_attention: the lengths add up to more rows than there are")
    if out is None:
        out, out_by = torch.empty_like(q, memory_format=torch.contiguous_format), -(-hq * D // 8) * 8
    else:
        out_rows, _, _, out_by = _bf16_rows("out", out, at, hq, D)
        if total > out_rows:
            raise ValueError("prompt_attention: out has fewer rows than q_lens")
    ql, kl = _ints(q_lens), _ints(k_lens)
    pq, pk = _addr(ql), _addr(kl)
    L = lib()
    need = L.swl_prompt_attention_part_floats(n, pq, pk, hq, hkv, D)
    part = torch.empty(need, dtype=torch.float32, device=at) if need > 0 else None
    check(L.swl_prompt_attention(n, pq, pk, q.data_ptr(), q_by, k.data_ptr(), k_by, v.data_ptr(), v_by, out.data_ptr(), out_by,
                                 hq, hkv, D, float(scale) if scale is not None else D ** -0.5,
                                 part.data_ptr() if part is not None else None, _current(at)))
    return out


def attention_device_error(device=None) -> int:
    """Synchronously reads and clears the bounded-wait error word of prompt_attention and
    paged_attention_kv4 on a device (default: the current one). Not 0: a wait inside a kernel ran
    out and outputs since the last reading may be wrong."""
    code = C.c_uint(0)
    with torch.cuda.device(device):
        check(lib().swl_attention_device_error(C.byref(code)))
    return int(code.value)


_KV4_BLOCK = {64: 1152, 128: 2304}  # swl_kv4_block_bytes


def kv4_block_bytes(head_dim: int = 128) -> int:
    """Bytes of one cache block: 16 tokens of one kv head, K and V."""
    n = _KV4_BLOCK.get(head_dim)
    if not n:
        raise ValueError(f"kv4 cache: head_dim must be 64 or 128 (got {head_dim})")
    return n


def kv4_cache(num_pages: int, hkv: int, head_dim: int = 128, page: int = 16, device=None) -> torch.Tensor:
    """An empty 4-bit cache: uint8 [num_pages, page / 16, hkv, block bytes]."""
    if page < 16 or page > 1024 or page & (page - 1):
        raise ValueError("kv4 cache: page must be 16, 32, 64 .. 1024 tokens")
    return torch.zeros(num_pages, page // 16, hkv, kv4_block_bytes(head_dim), dtype=torch.uint8,
                       device=device if device is not None else "cuda")


def _check_slots(what: str, t: torch.Tensor, n: int, dtype, at: int, dims: int) -> int:
    """One row per slot, contiguous inside; returns the rows' stride."""
    st = t.stride()
    if t.dtype is not dtype or t.get_device() != at or len(st) != dims or t.shape[0] != n or (st[-1] != 1 and t.shape[-1] > 1):
        raise ValueError(f"{what}: {dtype} on cuda:{at}, one row per slot, contiguous inside")
    return st[0]


def _slot_rows(ts, n: int, what: str, dtype, size: int, at: int, first=None) -> array:
    """Addresses of each slot's rows (elements of `size` bytes): a list of tensors,
    or one tensor with a row per slot (first: the first row of each slot)."""
    if isinstance(ts, torch.Tensor):
        if first is None:
            by = size * _check_slots(what, ts, n, dtype, at, ts.dim())
            first = range(n)
        else:
            by = size * ts.stride(0)
            if ts.dtype is not dtype or ts.get_device() != at or (ts.stride(-1) != 1 and ts.shape[-1] > 1):
                raise ValueError(f"{what}: {dtype} rows on cuda:{at}, contiguous inside")
        base = ts.data_ptr()
        return array("Q", [base + i * by for i in first])
    if len(ts) != n or any(t.dtype is not dtype or t.get_device() != at or
                           (t.dim() and t.numel() > 1 and t.stride(-1) != 1) for t in ts):
        raise ValueError(f"{what}: one {dtype} tensor per slot on cuda:{at}, contiguous inside")
    return array("Q", [t.data_ptr() for t in ts])


def _kv4_check(cache: torch.Tensor, hkv: int, head_dim: int, page: int, at: int) -> int:
    """A cache as kv4_cache makes it; returns its pages."""
    want = (page // 16, hkv, kv4_block_bytes(head_dim))
    shape = cache.shape
    if cache.dtype is not torch.uint8 or cache.get_device() != at or not cache.is_contiguous() or shape[1:] != want:
        raise ValueError(f"4-bit cache: contiguous uint8 [pages, {want[0]}, {want[1]}, {want[2]}] on cuda:{at} is needed")
    return shape[0]


def _kv4_slots(block_tables, caches, n: int, hkv: int, head_dim: int, page: int, at: int):
    """Block tables, their lengths, caches and their pages of a call over slots."""
    if isinstance(block_tables, torch.Tensor):
        if block_tables.dim() != 2:
            raise ValueError("block tables: [slots, pages] or one tensor per slot")
        lens = [block_tables.shape[1]] * n
    else:
        lens = [t.numel() for t in block_tables]
        if any(not t.dim() or t.shape[-1] != k for t, k in zip(block_tables, lens)):
            raise ValueError("block tables: one row of page ids per slot")
    tables = _slot_rows(block_tables, n, "block tables", torch.int32, 4, at)
    if isinstance(caches, torch.Tensor):
        caches = [caches] * n
    for c in {id(c): c for c in caches}.values():
        _kv4_check(c, hkv, head_dim, page, at)
    if len(caches) != n:
        raise ValueError("4-bit cache: one for all slots, or one per slot")
    return tables, _ints(lens), array("Q", [c.data_ptr() for c in caches]), array("q", [c.shape[0] for c in caches])


def _packed_slots(block_tables, caches, n: int, hkv: int, head_dim: int, page: int, at: int) -> tuple:
    """Of one table of block tables and one cache: the table, the elements between
    its rows and its length, the cache and its pages."""
    by = _check_slots("block tables", block_tables, n, torch.int32, at, 2)
    pages = _kv4_check(caches, hkv, head_dim, page, at)
    return block_tables.data_ptr(), by, block_tables.shape[1], caches.data_ptr(), pages


def _tensors(a, b) -> bool:
    return isinstance(a, torch.Tensor) and isinstance(b, torch.Tensor)


def _first_rows(rows) -> list:
    return [0, *itertools.accumulate(rows)][:len(rows)]


def _packed(name: str, t: torch.Tensor, rows: int, width: int, at: int) -> int:
    """Contiguous bf16 rows of `width` elements; returns their number."""
    have = t.shape[0]
    if t.dtype is not _BF16 or t.get_device() != at or not t.is_contiguous() or have < rows or t.numel() != have * width:
        raise ValueError(f"{name}: contiguous bf16 with at least {rows} rows of {width} on cuda:{at} is needed")
    return have


def _slots_of_rows(name: str, ts, rows, total: int, width: int) -> int:
    """Checks rows packed in one tensor or given per slot; returns their stride."""
    if isinstance(ts, torch.Tensor):
        shape = ts.shape
        if len(shape) != 2 or shape[1] < width or shape[0] < total:
            raise ValueError(f"{name}: {tuple(shape)} holds fewer than {total} rows of {width}")
        return _row_stride(ts)
    if len(ts) != len(rows) or any(t.dim() != 2 or t.shape[1] < width or t.shape[0] < r for t, r in zip(ts, rows)):
        raise ValueError(f"{name}: each slot must hold its rows of {width}")
    strides = {t.stride(0) for t in ts if t.shape[0] > 1}
    if len(strides) > 1:
        raise ValueError(f"{name}: the slots' rows must have one stride")
    return strides.pop() if strides else -(-width // 8) * 8


def kv4_append(qkvs, block_tables, caches, seqlens, q_rot, cos_sin, hq: int, hkv: int, head_dim: int = 128,
               page: int = 16, rows=None, k_rot=None, stream=None) -> None:
    """rope_append into a 4-bit cache: rotates the new rows' q and k (rotated q
    to q_rot [rows, hq * D], k to k_rot [rows, hkv * D] when given) and appends k
    and v quantised. qkvs: one tensor of rows per slot, or all rows packed
    in one tensor (then `rows` counts them per slot); block_tables: int32, one per
    slot (of any lengths) or [slots, pages]; caches: kv4_cache, one or one per slot (of
    any page counts); seqlens: int32, tokens cached before."""
    at = q_rot.get_device()
    if _elsewhere(at, stream):
        with _there(at, stream):
            return kv4_append(qkvs, block_tables, caches, seqlens, q_rot, cos_sin, hq, hkv, head_dim, page, rows, k_rot)
    packed = isinstance(qkvs, torch.Tensor)
    if rows is None:
        if packed:
            raise ValueError("kv4_append: packed rows need their counts")
        rows = [t.shape[0] for t in qkvs]
    n, total = len(rows), sum(rows)
    stride = _slots_of_rows("kv4_append: qkv", qkvs, rows, total, (hq + 2 * hkv) * head_dim)
    _packed("kv4_append: q_rot", q_rot, total, hq * head_dim, at)
    if k_rot is not None:
        _packed("kv4_append: k_rot", k_rot, total, hkv * head_dim, at)
    max_pos = _packed("kv4_append: cos_sin", cos_sin, 1, head_dim, at)
    counts = _ints(rows)
    tail = (hq, hkv, head_dim, page, cos_sin.data_ptr(), max_pos, q_rot.data_ptr(),
            k_rot.data_ptr() if k_rot is not None else None, _current(at))
    if n and packed and _tensors(block_tables, caches) and isinstance(seqlens, torch.Tensor):  # no tables of addresses to make
        if qkvs.dtype is not torch.bfloat16 or qkvs.get_device() != at or qkvs.stride()[1] != 1:
            raise ValueError(f"kv4_append: qkv: bf16 rows on cuda:{at} are needed")
        _check_slots("kv4_append: seqlens", seqlens, n, torch.int32, at, 1)
        slots = _packed_slots(block_tables, caches, n, hkv, head_dim, page, at)
        check(lib().swl_kv4_append_packed(n, _addr(counts), qkvs.data_ptr(), stride, *slots, seqlens.data_ptr(), *tail))
        return
    src = _slot_rows(qkvs, n, "kv4_append: qkv", torch.bfloat16, 2, at, _first_rows(rows) if packed else None)
    tables, table_lens, cache, pages = _kv4_slots(block_tables, caches, n, hkv, head_dim, page, at)
    lens = _slot_rows(seqlens, n, "kv4_append: seqlens", torch.int32, 4, at)
    check(lib().swl_kv4_append_each(n, _addr(counts), _addr(src), stride, _addr(tables), _addr(table_lens), _addr(cache),
                                    _addr(pages), _addr(lens), *tail))


def kv4_gather(block_tables, caches, starts, lens, k_out, v_out, hkv: int, head_dim: int = 128, page: int = 16,
               stream=None) -> None:
    """Tokens starts[i] .. starts[i] + lens[i] - 1 of each slot's 4-bit cache as
    packed bf16 rows of K and V (k_out, v_out [sum lens, hkv, D]): the keys
    that prompt_attention reads for a chunk behind a cached prefix."""
    at = k_out.get_device()
    if _elsewhere(at, stream):
        with _there(at, stream):
            return kv4_gather(block_tables, caches, starts, lens, k_out, v_out, hkv, head_dim, page)
    n, total = len(lens), sum(lens)
    if len(starts) != n:
        raise ValueError("kv4_gather: one start per slot is needed")
    _packed("kv4_gather: k_out", k_out, total, hkv * head_dim, at)
    _packed("kv4_gather: v_out", v_out, total, hkv * head_dim, at)
    begin, count = _ints(starts), _ints(lens)
    tail = (hkv, head_dim, page, k_out.data_ptr(), v_out.data_ptr(), _current(at))
    if n and _tensors(block_tables, caches):
        slots = _packed_slots(block_tables, caches, n, hkv, head_dim, page, at)
        check(lib().swl_kv4_gather_packed(n, _addr(begin), _addr(count), *slots, *tail))
        return
    tables, table_lens, cache, pages = _kv4_slots(block_tables, caches, n, hkv, head_dim, page, at)
    check(lib().swl_kv4_gather_each(n, _addr(begin), _addr(count), _addr(tables), _addr(table_lens), _addr(cache),
                                    _addr(pages), *tail))


def kv4_part_floats(rows, hq: int, hkv: int, max_len: int, head_dim: int = 128) -> int:
    """fp32 scratch values that paged_attention_kv4 needs for such a call."""
    counts = _ints(rows)
    return int(lib().swl_kv4_part_floats(len(rows), _addr(counts), hq, hkv, head_dim, max_len))


def paged_attention_kv4(rows, block_tables, caches, seqlens, outs, q_rot, hq: int, hkv: int, max_len: int, scale: float,
                        head_dim: int = 128, page: int = 16, part=None, stream=None) -> None:
    """paged_attention over a 4-bit cache: rows[i] new rows of slot i (already
    appended) at positions seqlens[i] + t. outs: one tensor of rows per slot,
    or all rows packed in one [rows, hq * D]. part: kv4_part_floats fp32 of scratch for
    this call alone (allocated here when None)."""
    at = q_rot.get_device()
    if _elsewhere(at, stream):
        with _there(at, stream):
            return paged_attention_kv4(rows, block_tables, caches, seqlens, outs, q_rot, hq, hkv, max_len, scale, head_dim,
                                       page, part)
    n, total, width = len(rows), sum(rows), hq * head_dim
    _packed("paged_attention_kv4: q_rot", q_rot, total, width, at)
    stride = _slots_of_rows("paged_attention_kv4: out", outs, rows, total, width)
    counts = _ints(rows)
    L = lib()
    need = L.swl_kv4_part_floats(n, _addr(counts), hq, hkv, head_dim, max_len)
    if part is None:
        if need > 0:
            part = torch.empty(need, dtype=torch.float32, device=at)
    elif part.dtype is not torch.float32 or part.get_device() != at or not part.is_contiguous() or part.numel() < need:
        raise ValueError(f"paged_attention_kv4: part needs {need} contiguous fp32 values on cuda:{at}")
    tail = (stride, hq, hkv, head_dim, page, float(scale), max_len, q_rot.data_ptr(),
            part.data_ptr() if part is not None else None, _current(at))
    if n and _tensors(block_tables, caches) and _tensors(seqlens, outs):
        if outs.dtype is not torch.bfloat16 or outs.get_device() != at or outs.stride()[1] != 1:
            raise ValueError(f"paged_attention_kv4: out: bf16 rows on cuda:{at} are needed")
        _check_slots("paged_attention_kv4: seqlens", seqlens, n, torch.int32, at, 1)
        slots = _packed_slots(block_tables, caches, n, hkv, head_dim, page, at)
        check(L.swl_paged_attention_kv4_packed(n, _addr(counts), *slots, seqlens.data_ptr(), outs.data_ptr(), *tail))
        return
    first = _first_rows(rows) if isinstance(outs, torch.Tensor) else None
    dst = _slot_rows(outs, n, "paged_attention_kv4: out", torch.bfloat16, 2, at, first)
    tables, table_lens, cache, pages = _kv4_slots(block_tables, caches, n, hkv, head_dim, page, at)
    lens = _slot_rows(seqlens, n, "paged_attention_kv4: seqlens", torch.int32, 4, at)
    check(L.swl_paged_attention_kv4_each(n, _addr(counts), _addr(tables), _addr(table_lens), _addr(cache), _addr(pages),
                                         _addr(lens), _addr(dst), *tail))


def rms_norm(xs, outs, w: torch.Tensor, eps: float, rows=None, x_stride: int | None = None,
             out_stride: int | None = None, stream=None) -> None:
    rows = rows if rows is not None else [int(x.shape[0]) for x in xs]
    x_stride = x_stride if x_stride is not None else int(xs[0].stride(0))
    out_stride = out_stride if out_stride is not None else int(outs[0].stride(0))
    check(lib().swl_rms_norm(len(xs), i32_array(rows), _ptrs(xs), x_stride, _ptrs(outs),
                             out_stride, w.data_ptr(), int(w.shape[0]), float(eps),
                             _stream(stream)))
