"""A KV cache in the model's 16 bits and the attention of decoded tokens over it.

The cache is a pool of pages of 64 tokens, keys and values [pages, KVH, 64, D] in fp16 or bf16.  Token i
of sequence b is row i % 64 of page ``block_table[b, i // 64]`` (int32; entries outside the pool name
no page): the tables and lengths are those of the 8-bit cache (``kv_int8``), whose half of the
bytes cost the keys' and values' bits.  ``kv_append`` writes keys that are rotated already, such as the
key states [B, KVH, S, 256] of ``prefix_attention``: ``kv_append(keys.transpose(1, 2), v.unflatten(-1, (KVH, 256)), ..)``,
views both; ``qk_norm_rope_append`` norms and rotates on the way;
``kv_attention`` attends decoded tokens over the cache, one a sequence or a few (action tokens behind a
prefix, drafts).  Lengths live on the device and are the caller's to advance.
"""

from __future__ import annotations

from collections.abc import Sequence

import torch

from pi05_fast.w4a4 import extension as _ext
from pi05_fast.w4a4.extension import (_changed, _check, _direct, _on_device, _ptr, _refuse_gradients, _refuse_tangents, _stream,
                                      _workspace, load_int4_gemm)
from pi05_fast.w4a4.int8 import ELEM
from pi05_fast.w4a4.kv_int8 import HEAD_DIMS, MAX_BATCH, MAX_TOKENS, PAGE_TOKENS, _ints
from pi05_fast.w4a4.rope import _check_rope, _heads, _meta, _plan, _strides, _weight

MAX_KV_HEADS = 32767


def _table_plan(table: torch.Tensor) -> tuple[int, int | None]:
    """Columns and row stride of a block table for the library (None: to be copied)."""
    rows, cols = table.shape
    if cols > 1 and table.stride(1) != 1:
        return cols, None
    return cols, table.stride(0) if rows > 1 else cols


def kv_cache(pages: int, kv_heads: int, head_dim: int, dtype: torch.dtype, device) -> tuple[torch.Tensor, torch.Tensor]:
    """An empty pool: (k_cache, v_cache)."""
    if head_dim not in HEAD_DIMS:
        raise RuntimeError(f"the KV cache takes head_dim 64, 128 or 256, got {head_dim}")
    if dtype not in ELEM:
        raise RuntimeError(f"the KV cache holds float16 or bfloat16, got {dtype}")
    shape = (pages, kv_heads, PAGE_TOKENS, head_dim)
    return torch.zeros(shape, dtype=dtype, device=device), torch.zeros(shape, dtype=dtype, device=device)


def _check_cache(what, x, k_cache, v_cache, table, lens, b, t, kvh, d):
    dev = x.device
    if d not in HEAD_DIMS:
        raise RuntimeError(f"{what}: head_dim must be 64, 128 or 256, got {d}")
    pages = k_cache.size(0) if k_cache.dim() else 0
    for name, c in (("k_cache", k_cache), ("v_cache", v_cache)):
        if c.dtype != x.dtype or c.shape != (pages, kvh, PAGE_TOKENS, d):
            raise RuntimeError(f"{what}: {name} must be {x.dtype} [pages, {kvh}, {PAGE_TOKENS}, {d}], got {c.dtype} {tuple(c.shape)}")
    if table.dtype != torch.int32 or table.dim() != 2 or table.size(0) != b:
        raise RuntimeError(f"{what}: block_table must be int32 [{b}, pages of a sequence], got {table.dtype} "
                           f"{tuple(table.shape)}")
    # Here: the library takes them as 32 bits.
    if b > MAX_BATCH or t > MAX_TOKENS or table.size(1) > MAX_TOKENS or kvh > MAX_KV_HEADS or pages > 0x7fffffff:
        raise RuntimeError(f"{what}: at most {MAX_BATCH} sequences, {MAX_TOKENS} tokens and {MAX_TOKENS} pages of a sequence, "
                           f"{MAX_KV_HEADS} KV heads and 2^31 - 1 pages, got {b}, {t}, {table.size(1)}, {kvh} and {pages}")
    if lens.dtype != torch.int32 or lens.shape != (b,):
        raise RuntimeError(f"{what}: lens must be int32 [{b}], got {lens.dtype} {tuple(lens.shape)}")
    for c in (k_cache, v_cache, table, lens):
        if c.device != dev:
            raise RuntimeError(f"{what}: the cache, block_table and lens must be on {dev}, got {c.device}")
    if not (k_cache.is_contiguous() and v_cache.is_contiguous()):
        raise RuntimeError(f"{what}: the cache must be contiguous")
    return pages


def _check_append(what, k, v, k_cache, v_cache, table, lens, counts):
    if not k.is_cuda:
        raise RuntimeError(f"{what} expects CUDA/HIP tensors")
    elem = ELEM.get(k.dtype)
    if elem is None or v.dtype != k.dtype:
        raise RuntimeError(f"{what} takes float16 or bfloat16 keys and values of one type, got {k.dtype} and {v.dtype}")
    if k.dim() != 4 or v.shape != k.shape or v.device != k.device:
        raise RuntimeError(f"{what} expects k and v [B, T, KVH, D] on one device, got {tuple(k.shape)} and {tuple(v.shape)}")
    b, t, kvh, d = k.shape
    pages = _check_cache(what, k, k_cache, v_cache, table, lens, b, t, kvh, d)
    _ints(what, "counts", counts, b, k.device)
    if b * t > MAX_TOKENS:  # here: the library takes them as 32 bits
        raise RuntimeError(f"{what}: at most {MAX_TOKENS} tokens a call, got {b} x {t}")
    return (elem, b, t, kvh, d), pages, _strides(k), _strides(v), *_table_plan(table)


def _cache_pointers(what, k_cache, v_cache):
    kp, vp = k_cache.data_ptr(), v_cache.data_ptr()
    if (kp | vp) & 15:
        raise RuntimeError(f"{what}: the cache must be 16-byte aligned")
    return kp, vp


def _append_impl(k, v, k_cache, v_cache, block_table, lens, counts):
    what = "kv_append"
    shape, pages, ks, vs, cols, stride = _plan(
        (what, k.dtype, k.device, k.shape, k.stride(), v.dtype, v.device, v.shape, v.stride(), k_cache.dtype, k_cache.device, k_cache.shape,
         k_cache.stride(), v_cache.dtype, v_cache.device, v_cache.shape, v_cache.stride(), block_table.dtype, block_table.device,
         block_table.shape, block_table.stride(), lens.dtype, lens.device, lens.shape, _meta(counts)),
        lambda: _check_append(what, k, v, k_cache, v_cache, block_table, lens, counts))
    kp, vp = _cache_pointers(what, k_cache, v_cache)
    if shape[1] == 0 or shape[2] == 0:
        return
    dev = k.device
    table = block_table
    if stride is None:
        table, stride = table.contiguous(), cols
    lens, counts = lens.contiguous(), None if counts is None else counts.contiguous()
    k, ks = _heads(k, ks)
    v, vs = _heads(v, vs)
    lib = _ext._lib if _ext._lib is not None else load_int4_gemm()
    with _on_device(dev):
        _check(lib.pi05w4a4_kv_append(k.data_ptr(), ks, v.data_ptr(), vs, *shape, kp, vp, pages, table.data_ptr(), stride,
                                      cols, lens.data_ptr(), _ptr(counts), _stream(dev)), "pi05w4a4_kv_append")


def _check_rope_append(what, q, k, v, q_weight, k_weight, positions, inv_freq, k_cache, v_cache, table, lens, counts, axes):
    found = _check_rope(what, q, k, q_weight, k_weight, positions, inv_freq, axes)
    if v.dtype != k.dtype or v.shape != k.shape or v.device != q.device:
        raise RuntimeError(f"{what}: v must be {k.dtype} {tuple(k.shape)} on {q.device}, got {v.dtype} {tuple(v.shape)} on {v.device}")
    _, b, t, _, kvh, d = found[0]
    pages = _check_cache(what, q, k_cache, v_cache, table, lens, b, t, kvh, d)
    _ints(what, "counts", counts, b, q.device)
    return *found, pages, _strides(v), *_table_plan(table)


def _rope_append_impl(q, k, v, q_weight, k_weight, eps, positions, inv_freq, k_cache, v_cache, block_table, lens, counts,
                      unit_offset, interleaved, axes):
    what = "qk_norm_rope_append"
    axes = None if axes is None else tuple(axes)
    shape, qs, ks, ps, pos_bytes, count, amap, rot, pages, vs, cols, stride = _plan(
        (what, axes, q.dtype, q.device, q.shape, q.stride(), k.dtype, k.device, k.shape, k.stride(), v.dtype, v.device, v.shape, v.stride(),
         _meta(q_weight), _meta(k_weight), positions.dtype, positions.device, positions.shape, positions.stride(), inv_freq.dtype,
         inv_freq.device, inv_freq.shape, k_cache.dtype, k_cache.device, k_cache.shape, k_cache.stride(), v_cache.dtype, v_cache.device,
         v_cache.shape, v_cache.stride(), block_table.dtype, block_table.device, block_table.shape, block_table.stride(), lens.dtype,
         lens.device, lens.shape, _meta(counts)),
        lambda: _check_rope_append(what, q, k, v, q_weight, k_weight, positions, inv_freq, k_cache, v_cache, block_table, lens,
                                   counts, axes))
    kp, vp = _cache_pointers(what, k_cache, v_cache)
    dev = q.device
    q_out = torch.empty_like(q, memory_format=torch.contiguous_format)
    table = block_table
    if stride is None:
        table, stride = table.contiguous(), cols
    lens, counts = lens.contiguous(), None if counts is None else counts.contiguous()
    q, qs = _heads(q, qs)
    k, ks = _heads(k, ks)
    v, vs = _heads(v, vs)
    q_weight, k_weight, inv_freq = _weight(q_weight), _weight(k_weight), inv_freq.contiguous()
    lib = _ext._lib if _ext._lib is not None else load_int4_gemm()
    with _on_device(dev):
        _check(lib.pi05w4a4_qk_norm_rope_append(q.data_ptr(), qs, k.data_ptr(), ks, v.data_ptr(), vs, *shape, _ptr(q_weight),
                                                _ptr(k_weight), eps, unit_offset, positions.data_ptr(), ps, pos_bytes, count, amap,
                                                inv_freq.data_ptr(), rot, interleaved, q_out.data_ptr(), kp, vp, pages,
                                                table.data_ptr(), stride, cols, lens.data_ptr(), _ptr(counts), _stream(dev)),
               "pi05w4a4_qk_norm_rope_append")
    return q_out


def _check_attention(what, q, k_cache, v_cache, table, lens, q_lens):
    if not q.is_cuda:
        raise RuntimeError(f"{what} expects CUDA/HIP tensors")
    elem = ELEM.get(q.dtype)
    if elem is None:
        raise RuntimeError(f"{what} takes float16 or bfloat16 queries, got {q.dtype}")
    if q.dim() != 4 or k_cache.dim() != 4:
        raise RuntimeError(f"{what} expects q [B, T, H, D] and k_cache [pages, KVH, 64, D], got {tuple(q.shape)} and "
                           f"{tuple(k_cache.shape)}")
    b, t, h, d = q.shape
    kvh = k_cache.size(1)
    if kvh == 0 or h == 0 or h % kvh:
        raise RuntimeError(f"{what}: the query heads must be a multiple of the KV heads, got {h} and {kvh}")
    if h > 65535:  # here: the library takes them as 32 bits
        raise RuntimeError(f"{what}: at most 65535 query heads, got {h}")
    pages = _check_cache(what, q, k_cache, v_cache, table, lens, b, t, kvh, d)
    _ints(what, "q_lens", q_lens, b, q.device)
    with _on_device(q.device):
        need = int(load_int4_gemm().pi05w4a4_kv_attention_workspace_bytes(b, t, h, kvh, d, table.size(1)))
    return (elem, b, t, h, kvh, d), pages, _strides(q), need, *_table_plan(table)


def _attention_impl(q, k_cache, v_cache, block_table, lens, scaling, causal, q_lens, return_lse):
    what = "kv_attention"
    shape, pages, qs, need, cols, stride = _plan(
        (what, q.dtype, q.device, q.shape, q.stride(), k_cache.dtype, k_cache.device, k_cache.shape, k_cache.stride(), v_cache.dtype,
         v_cache.device, v_cache.shape, v_cache.stride(), block_table.dtype, block_table.device, block_table.shape, block_table.stride(),
         lens.dtype, lens.device, lens.shape, _meta(q_lens)),
        lambda: _check_attention(what, q, k_cache, v_cache, block_table, lens, q_lens))
    kp, vp = _cache_pointers(what, k_cache, v_cache)
    dev = q.device
    out = torch.empty_like(q, memory_format=torch.contiguous_format)
    lse = torch.empty(q.shape[:3], dtype=torch.float32, device=dev) if return_lse else None
    if shape[1] == 0 or shape[2] == 0:
        return out, lse
    table = block_table
    if stride is None:
        table, stride = table.contiguous(), cols
    lens, q_lens = lens.contiguous(), None if q_lens is None else q_lens.contiguous()
    q, qs = _heads(q, qs)
    lib = _ext._lib if _ext._lib is not None else load_int4_gemm()
    with _on_device(dev):
        ws = _workspace(dev, need) if need else None
        _check(lib.pi05w4a4_kv_attention(q.data_ptr(), qs, *shape, kp, vp, pages, table.data_ptr(), stride, cols,
                                         lens.data_ptr(), _ptr(q_lens), scaling, causal, out.data_ptr(), _ptr(lse), _ptr(ws), need,
                                         _stream(dev)), "pi05w4a4_kv_attention")
    return out, lse


# ----------------------------------------------------------------------------- custom ops
@torch.library.custom_op("pi05_w4a4::kv_append", mutates_args=("k_cache", "v_cache"))
def _append_op(k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, block_table: torch.Tensor,
               lens: torch.Tensor, counts: torch.Tensor | None) -> None:
    _refuse_tangents(k, v, k_cache, v_cache)
    _append_impl(k, v, k_cache, v_cache, block_table, lens, counts)


@_append_op.register_fake
def _append_fake(k, v, k_cache, v_cache, block_table, lens, counts):
    return None


@torch.library.custom_op("pi05_w4a4::qk_norm_rope_append", mutates_args=("k_cache", "v_cache"))
def _rope_append_op(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, q_weight: torch.Tensor | None,
                    k_weight: torch.Tensor | None, eps: float, positions: torch.Tensor, inv_freq: torch.Tensor,
                    k_cache: torch.Tensor, v_cache: torch.Tensor, block_table: torch.Tensor, lens: torch.Tensor,
                    counts: torch.Tensor | None, unit_offset: bool, interleaved: bool,
                    axes: Sequence[int] | None) -> torch.Tensor:
    _refuse_tangents(q, k, v, q_weight, k_weight, inv_freq, k_cache, v_cache)
    return _rope_append_impl(q, k, v, q_weight, k_weight, eps, positions, inv_freq, k_cache, v_cache, block_table, lens, counts,
                             unit_offset, interleaved, axes)


@_rope_append_op.register_fake
def _rope_append_fake(q, k, v, q_weight, k_weight, eps, positions, inv_freq, k_cache, v_cache, block_table, lens, counts,
                      unit_offset, interleaved, axes):
    return q.new_empty(q.shape)


@torch.library.custom_op("pi05_w4a4::kv_attention", mutates_args=())
def _attention_op(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, block_table: torch.Tensor,
                  lens: torch.Tensor, scaling: float, causal: bool, q_lens: torch.Tensor | None,
                  return_lse: bool) -> tuple[torch.Tensor, torch.Tensor]:
    _refuse_tangents(q, k_cache, v_cache)
    out, lse = _attention_impl(q, k_cache, v_cache, block_table, lens, scaling, causal, q_lens, return_lse)
    return out, lse if lse is not None else out.new_empty((0,), dtype=torch.float32)


@_attention_op.register_fake
def _attention_fake(q, k_cache, v_cache, block_table, lens, scaling, causal, q_lens, return_lse):
    return q.new_empty(q.shape), q.new_empty(q.shape[:-1] if return_lse else (0,), dtype=torch.float32)


# ----------------------------------------------------------------------------- public functions
def kv_append(k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, block_table: torch.Tensor,
              lens: torch.Tensor, counts: torch.Tensor | None = None) -> None:
    """Write k and v [B, T, KVH, D] (the cache's type, any strides) behind each sequence's ``lens`` [B]
    cached tokens, the first ``counts`` [B] of them (None: all T); the rest of a padded batch is
    not written.  Changes those rows of the cache and nothing else, and leaves ``lens`` as it is.
    Tokens past the table, or whose table entry names no page, are dropped.  Full pages can be
    shared between sequences; a row may be written from one place of a call only.  k and v must not lie
    in the cache.  There are no derivatives: arguments that require gradients are refused."""
    if _direct(k, v, k_cache, v_cache, block_table, lens, counts):
        _append_impl(k, v, k_cache, v_cache, block_table, lens, counts)
        return _changed((k_cache, v_cache))
    _refuse_gradients("kv_append", k, v, k_cache, v_cache)
    return torch.ops.pi05_w4a4.kv_append(k, v, k_cache, v_cache, block_table, lens, counts)


def qk_norm_rope_append(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, q_weight: torch.Tensor | None,
                        k_weight: torch.Tensor | None, eps: float, positions: torch.Tensor, inv_freq: torch.Tensor,
                        k_cache: torch.Tensor, v_cache: torch.Tensor, block_table: torch.Tensor, lens: torch.Tensor,
                        counts: torch.Tensor | None = None, unit_offset: bool = True, interleaved: bool = False,
                        axes: Sequence[int] | None = None) -> torch.Tensor:
    """``qk_norm_rope`` of q and k and ``kv_append`` of the rotated keys and of v in one launch: returns
    the queries [B, T, H, D].  ``positions`` are the tokens' own (with several axes they are not the
    places in the cache, which follow from ``lens``).  All T tokens' queries are computed; keys and
    values go into the cache up to ``counts``.  There are no derivatives: arguments that require
    gradients are refused."""
    if _direct(q, k, v, q_weight, k_weight, positions, inv_freq, k_cache, v_cache, block_table, lens, counts):
        q_out = _rope_append_impl(q, k, v, q_weight, k_weight, float(eps), positions, inv_freq, k_cache, v_cache, block_table, lens,
                                  counts, bool(unit_offset), bool(interleaved), axes)
        _changed((k_cache, v_cache))
        return q_out
    _refuse_gradients("qk_norm_rope_append", q, k, v, q_weight, k_weight, inv_freq, k_cache, v_cache)
    return torch.ops.pi05_w4a4.qk_norm_rope_append(q, k, v, q_weight, k_weight, float(eps), positions, inv_freq, k_cache, v_cache,
                                                   block_table, lens, counts, bool(unit_offset), bool(interleaved),
                                                   None if axes is None else list(axes))


def kv_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, block_table: torch.Tensor, lens: torch.Tensor,
                 scaling: float, causal: bool = True, q_lens: torch.Tensor | None = None, return_lse: bool = False):
    """softmax(scaling q K^T) V of q [B, T, H, D] (the cache's type, rotated, any strides) over the
    cache: [B, T, H, D].  H is a multiple of KVH; query head h reads KV head h // (H / KVH).  Made for
    decoded tokens, T = 1 or a few: every 16 rows of T * (H / KVH), 64 where rows are many, read the cache once.  The work is planned
    for the table's width: pass a table held at capacity as ``block_table[:, :n]``, n the pages of
    the longest sequence.  Entries that name no page hide their 64 tokens.

    The queries are the last T tokens (``q_lens`` [B]: the last q_lens[b], the rows behind them
    padding) of ``lens`` [B] cached ones, whose keys the cache holds already.  When ``causal``, query i
    sees the first lens - q_len + i + 1 tokens, else all of them.  A length past the table (64 tokens an
    entry) counts as the table's, for the place of the queries too.  A query that sees no token, a
    padding row among them, gets zeros, and so does one whose scores are all minus infinity.  What a query does not see has no effect on it, whatever it
    holds; a NaN or infinity among the values it sees makes its output in that dimension NaN or infinite.  With
    ``return_lse``, also the natural log of the sum of exp(scaling q k), fp32 [B, T, H] (-inf where none
    is seen), with which attention over further keys can be joined."""
    if _direct(q, k_cache, v_cache, block_table, lens, q_lens):
        out, lse = _attention_impl(q, k_cache, v_cache, block_table, lens, float(scaling), bool(causal), q_lens, bool(return_lse))
    else:
        out, lse = torch.ops.pi05_w4a4.kv_attention(q, k_cache, v_cache, block_table, lens, float(scaling), bool(causal), q_lens,
                                                    bool(return_lse))
    return (out, lse) if return_lse else out
