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

import ctypes as C
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
def _bf16_rows(name: str, t: torch.Tensor, heads: int | None, head_dim: int | None, device=None) -> None:
    """A bf16 CUDA tensor [rows, heads, head_dim] whose heads are contiguous."""
    if t.dtype != torch.bfloat16 or not t.is_cuda or (device is not None and t.device != device):
        raise ValueError(f"{name}: a bf16 tensor on the call's CUDA device is needed")
    if t.dim() != 3 or (heads is not None and t.shape[1] != heads) or (head_dim is not None and t.shape[2] != head_dim):
        raise ValueError(f"{name}: shape {tuple(t.shape)} does not fit")
    if t.numel() and (t.stride(2) != 1 or (t.shape[1] > 1 and t.stride(1) != t.shape[2])):
        raise ValueError(f"{name}: heads must be contiguous")


def _row_stride(t: torch.Tensor) -> int:
    """Elements between rows; a single row's stride is never used (torch leaves it arbitrary)."""
    width = t.shape[-1] * (t.shape[-2] if t.dim() == 3 else 1)
    return int(t.stride(0)) if t.shape[0] > 1 else -(-width // 8) * 8


def prompt_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, q_lens, k_lens=None, scale: float | None = None,
                     out: torch.Tensor | None = None, stream=None) -> torch.Tensor:
    """Causal GQA attention of packed sequences: q [sum q_lens, hq, D], k and v
    [sum k_lens, hkv, D] (row-strided views allowed), lengths on the host. Row
    r of a sequence sees its keys 0 .. r + k_len - q_len (k_lens defaults to
    q_lens; longer ones hold a prefix); a row without keys gives zeros.
    Returns out [rows of q, hq, D] (rows behind the last sequence are left as they are)."""
    _bf16_rows("q", q, None, None)
    hq, D = int(q.shape[1]), int(q.shape[2])
    _bf16_rows("k", k, None, D, q.device)
    hkv = int(k.shape[1])
    _bf16_rows("v", v, hkv, D, q.device)
    q_lens = [int(x) for x in q_lens]
    k_lens = q_lens if k_lens is None else [int(x) for x in k_lens]
    if len(k_lens) != len(q_lens):
        raise ValueError("prompt_attention: one key length per sequence")
    if sum(q_lens) > q.shape[0] or sum(k_lens) > min(k.shape[0], v.shape[0]):
        raise ValueError("prompt_attention: the lengths add up to more rows than there are")
    n, ql, kl = len(q_lens), i32_array(q_lens), i32_array(k_lens)
    with torch.cuda.device(q.device):
        s = stream if stream is not None else torch.cuda.current_stream()
        with torch.cuda.stream(s):  # the scratch belongs to the stream that uses it
            if out is None:
                out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
            else:
                _bf16_rows("out", out, hq, D, q.device)
                if sum(q_lens) > out.shape[0]:
                    raise ValueError("prompt_attention: out has fewer rows than q_lens")
            need = int(lib().swl_prompt_attention_part_floats(n, ql, kl, hq, hkv, D))
            part = torch.empty(need, dtype=torch.float32, device=q.device) if need > 0 else None
            check(lib().swl_prompt_attention(n, ql, kl, q.data_ptr(), _row_stride(q), k.data_ptr(), _row_stride(k),
                                             v.data_ptr(), _row_stride(v), out.data_ptr(), _row_stride(out), hq, hkv, D,
                                             float(scale) if scale is not None else D ** -0.5,
                                             part.data_ptr() if part is not None else None, s.cuda_stream))
    return out


def kv4_block_bytes(head_dim: int = 128) -> int:
    """Bytes of one cache block: 16 tokens of one kv head, K and V."""
    n = int(lib().swl_kv4_block_bytes(head_dim))
    if not n:
        raise ValueError(f"kv4 cache: head_dim must be 64 or 128 (got {head_dim})")
    return n


def kv4_cache(num_pages: int, hkv: int, head_dim: int = 128, page: int = 16, device=None) -> torch.Tensor:
    """An empty 4-bit cache: uint8 [num_pages, page / 16, hkv, block bytes]."""
    if page < 16 or page > 1024 or page & (page - 1):
        raise ValueError("kv4 cache: page must be 16, 32, 64 .. 1024 tokens")
    return torch.zeros(num_pages, page // 16, hkv, kv4_block_bytes(head_dim), dtype=torch.uint8,
                       device=device if device is not None else "cuda")


def _rows_of(ts, n: int, what: str, dtype, device, step=None) -> list:
    """Addresses of each slot's rows: a list of tensors, or one tensor with a
    row per slot (step: the first row of each slot)."""
    if isinstance(ts, torch.Tensor):
        if ts.dtype != dtype or ts.device != device:
            raise ValueError(f"{what}: {dtype} on {device} is needed")
        if (ts.dim() > 1 and ts.stride(-1) != 1) or (step is None and ts.shape[0] != n):
            raise ValueError(f"{what}: one row per slot, contiguous inside")
        base, by = ts.data_ptr(), ts.element_size() * int(ts.stride(0))
        return [base + i * by for i in (step if step is not None else range(n))]
    if len(ts) != n or any(t.dtype != dtype or t.device != device or (t.dim() and t.numel() > 1 and t.stride(-1) != 1)
                           for t in ts):
        raise ValueError(f"{what}: one {dtype} tensor per slot on {device}, contiguous inside")
    return [t.data_ptr() for t in ts]


def _kv4_slots(block_tables, caches, n: int, hkv: int, head_dim: int, page: int, device):
    """Block tables, their length, caches and their pages of a call over slots."""
    block = kv4_block_bytes(head_dim)
    if isinstance(block_tables, torch.Tensor):
        if block_tables.dim() != 2:
            raise ValueError("block tables: [slots, pages] or one tensor per slot")
        table_len = int(block_tables.shape[1])
    else:
        table_len = min((int(t.shape[0]) for t in block_tables), default=1)
    tables = _rows_of(block_tables, n, "block tables", torch.int32, device)
    each = [caches] if isinstance(caches, torch.Tensor) else list(caches)
    for c in each:
        if c.dtype != torch.uint8 or c.device != device or not c.is_contiguous() or \
                tuple(c.shape[1:]) != (page // 16, hkv, block):
            raise ValueError(f"4-bit cache: contiguous uint8 [pages, {page // 16}, {hkv}, {block}] on {device} is needed")
    ptrs = [caches.data_ptr()] * n if isinstance(caches, torch.Tensor) else [c.data_ptr() for c in each]
    if len(ptrs) != n:
        raise ValueError("4-bit cache: one for all slots, or one per slot")
    return ptr_array(tables), table_len, ptr_array(ptrs), min((int(c.shape[0]) for c in each), default=1)


def _first_rows(rows) -> list:
    out, at = [], 0
    for r in rows:
        out.append(at)
        at += r
    return out


def _packed(name: str, t: torch.Tensor, rows: int, width: int, device) -> None:
    if t.dtype != torch.bfloat16 or t.device != device or not t.is_contiguous() or t.shape[0] < rows or \
            t.numel() != t.shape[0] * width:
        raise ValueError(f"{name}: contiguous bf16 with at least {rows} rows of {width} on {device} is needed")


def kv4_append(qkvs, block_tables, caches, seqlens, q_rot, cos_sin, hq: int, hkv: int, head_dim: int = 128,
               page: int = 16, rows=None, k_rot=None, stream=None) -> None:
    """rope_append into a 4-bit cache: rotates the new rows' q and k (rotated q
    to q_rot [rows, hq * D], k to k_rot [rows, hkv * D] when given) and appends k
    and v quantised. qkvs: one tensor of rows per slot, or all rows packed
    in one tensor (then `rows` counts them per slot); block_tables: int32, one per slot or [slots, pages];
    caches: kv4_cache, one or one per slot; seqlens: int32, tokens cached before."""
    packed = isinstance(qkvs, torch.Tensor)
    if rows is None:
        if packed:
            raise ValueError("kv4_append: packed rows need their counts")
        rows = [int(t.shape[0]) for t in qkvs]
    rows = [int(r) for r in rows]
    n, total, dev = len(rows), sum(rows), q_rot.device
    width = (hq + 2 * hkv) * head_dim
    if dev.type != "cuda":
        raise ValueError("kv4_append: CUDA tensors are needed")
    if packed:
        if qkvs.dim() != 2 or qkvs.shape[1] < width or qkvs.shape[0] < total:
            raise ValueError(f"kv4_append: qkv {tuple(qkvs.shape)} holds fewer than {total} rows of {width}")
        stride = _row_stride(qkvs)
    else:
        if any(t.dim() != 2 or t.shape[1] < width or t.shape[0] < r for t, r in zip(qkvs, rows)):
            raise ValueError(f"kv4_append: each slot's qkv must hold its rows of {width}")
        strides = {_row_stride(t) for t in qkvs if t.shape[0] > 1} or {-(-width // 8) * 8}
        if len(strides) > 1:
            raise ValueError("kv4_append: the slots' rows must have one stride")
        stride = strides.pop()
    _packed("kv4_append: q_rot", q_rot, total, hq * head_dim, dev)
    if k_rot is not None:
        _packed("kv4_append: k_rot", k_rot, total, hkv * head_dim, dev)
    _packed("kv4_append: cos_sin", cos_sin, 1, head_dim, dev)
    src = _rows_of(qkvs, n, "kv4_append: qkv", torch.bfloat16, dev, _first_rows(rows) if packed else None)
    tables, table_len, cache, pages = _kv4_slots(block_tables, caches, n, hkv, head_dim, page, dev)
    lens = _rows_of(seqlens, n, "kv4_append: seqlens", torch.int32, dev)
    with torch.cuda.device(dev):
        check(lib().swl_kv4_append(n, i32_array(rows), ptr_array(src), stride, tables, table_len, cache, pages,
                                   ptr_array(lens), hq, hkv, head_dim, page, cos_sin.data_ptr(), int(cos_sin.shape[0]),
                                   q_rot.data_ptr(), k_rot.data_ptr() if k_rot is not None else None, _stream(stream)))


def kv4_gather(block_tables, caches, starts, lens, k_out, v_out, hkv: int, head_dim: int = 128, page: int = 16,
               stream=None) -> None:
    """Tokens starts[i] .. starts[i] + lens[i] - 1 of each slot's 4-bit cache as
    packed bf16 rows of K and V (k_out, v_out [sum lens, hkv, D]): the keys
    that prompt_attention reads for a chunk behind a cached prefix."""
    lens = [int(x) for x in lens]
    n, dev = len(lens), k_out.device
    if dev.type != "cuda" or len(starts) != n:
        raise ValueError("kv4_gather: CUDA tensors and one start per slot are needed")
    for name, t in (("k_out", k_out), ("v_out", v_out)):
        _packed(f"kv4_gather: {name}", t, sum(lens), hkv * head_dim, dev)
    tables, table_len, cache, pages = _kv4_slots(block_tables, caches, n, hkv, head_dim, page, dev)
    with torch.cuda.device(dev):
        check(lib().swl_kv4_gather(n, i32_array(starts), i32_array(lens), tables, table_len, cache, pages, hkv, head_dim,
                                   page, k_out.data_ptr(), v_out.data_ptr(), _stream(stream)))


def kv4_part_floats(rows, hq: int, hkv: int, max_len: int, head_dim: int = 128) -> int:
    return int(lib().swl_kv4_part_floats(len(rows), i32_array(rows), hq, hkv, head_dim, max_len))


def paged_attention_kv4(rows, block_tables, caches, seqlens, outs, q_rot, hq: int, hkv: int, max_len: int, scale: float,
                        head_dim: int = 128, page: int = 16, part=None, stream=None) -> None:
    """paged_attention over a 4-bit cache: rows[i] new rows of slot i (already
    appended) at positions seqlens[i] + t. outs: one tensor of rows per slot,
    or all rows packed in one [rows, hq * D]. part: kv4_part_floats fp32 of scratch for
    this call alone (allocated here when None)."""
    rows = [int(r) for r in rows]
    n, total, dev = len(rows), sum(rows), q_rot.device
    if dev.type != "cuda":
        raise ValueError("paged_attention_kv4: CUDA tensors are needed")
    _packed("paged_attention_kv4: q_rot", q_rot, total, hq * head_dim, dev)
    width = hq * head_dim
    packed = isinstance(outs, torch.Tensor)
    for t, r in [(outs, total)] if packed else zip(outs, rows):
        if t.dim() != 2 or t.shape[1] < width or t.shape[0] < r:
            raise ValueError(f"paged_attention_kv4: an output holds fewer than {r} rows of {width}")
    strides = {_row_stride(t) for t in ([outs] if packed else outs) if t.shape[0] > 1} or {-(-width // 8) * 8}
    if len(strides) > 1:
        raise ValueError("paged_attention_kv4: the slots' rows must have one stride")
    dst = _rows_of(outs, n, "paged_attention_kv4: out", torch.bfloat16, dev, _first_rows(rows) if packed else None)
    tables, table_len, cache, pages = _kv4_slots(block_tables, caches, n, hkv, head_dim, page, dev)
    lens = _rows_of(seqlens, n, "paged_attention_kv4: seqlens", torch.int32, dev)
    c_rows = i32_array(rows)
    need = int(lib().swl_kv4_part_floats(n, c_rows, hq, hkv, head_dim, max_len))
    with torch.cuda.device(dev):
        s = stream if stream is not None else torch.cuda.current_stream()
        if part is None and need > 0:
            with torch.cuda.stream(s):  # the scratch belongs to the stream that uses it
                part = torch.empty(need, dtype=torch.float32, device=dev)
        elif part is not None and (part.dtype != torch.float32 or part.device != dev or not part.is_contiguous() or
                                   part.numel() < need):
            raise ValueError(f"paged_attention_kv4: part needs {need} contiguous fp32 values on {dev}")
        check(lib().swl_paged_attention_kv4(n, c_rows, tables, table_len, cache, pages, ptr_array(lens), ptr_array(dst),
                                            strides.pop(), hq, hkv, head_dim, page, float(scale), max_len,
                                            q_rot.data_ptr(), part.data_ptr() if part is not None else None,
                                            s.cuda_stream))


def rms_norm(xs, outs, w: torch.Tensor, eps: float, rows=None, x_stride: int | None = None,
             out_stride: int | None = None, stream=None) -> None:
    rows = rows if rows is not None else [int(x.shape[0]) for x in xs]
    x_stride = x_stride if x_stride is not None else int(xs[0].stride(0))
    out_stride = out_stride if out_stride is not None else int(outs[0].stride(0))
    check(lib().swl_rms_norm(len(xs), i32_array(rows), _ptrs(xs), x_stride, _ptrs(outs),
                             out_stride, w.data_ptr(), int(w.shape[0]), float(eps),
                             _stream(stream)))
