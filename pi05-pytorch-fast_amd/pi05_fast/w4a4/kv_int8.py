"""A KV cache in 8 bits and the attention over it.

The cache is a pool of pages of 64 tokens: K codes int8 [pages, KVH, 64, D], V codes int8 [pages,
KVH, D, 64] (transposed within the page), and an fp32 scale for each page and KV head of either.
Token i of sequence b is row i % 64 of page ``block_table[b, i // 64]`` (int32; entries outside
the pool name no page).  ``int8_kv_append`` quantizes new keys (RoPE applied, as
``prefix_attention`` returns its key states) and values into it, ``int8_kv_attention`` attends
queries over it: decoded tokens, the action tokens behind a prefix, or a prompt's next chunk.

Half the bytes of an fp16 cache.  A page's scale is that of its largest value; where a later
token raises it, the page's earlier codes are rounded again (half a step of the new scale at
most), so that a page filled token by token is up to about 1.4 times as far from its values as
one written at once.  The scale does not fall again while the page keeps tokens: tokens that are
written over and over at one length leave it at the largest they ever needed.  Lengths live on the
device and are the caller's to advance.
"""

from __future__ import annotations

import ctypes

import torch

from pi05_fast.w4a4 import extension as _ext
from pi05_fast.w4a4.extension import (_changed, _check, _direct, _on_device, _ptr, _refuse_tangents, _stream, _workspace,
                                      load_int4_gemm)
from pi05_fast.w4a4.int8 import ELEM

PAGE_TOKENS = 64
HEAD_DIMS = (64, 128, 256)
MAX_BATCH = 65535
MAX_TOKENS = 1 << 24  # tokens of a sequence in a call, and pages of a table row

_STRIDES: dict[tuple, ctypes.Array] = {}
_ATTN_WS: dict[tuple, int] = {}


def int8_kv_cache(pages: int, kv_heads: int, head_dim: int, device) -> tuple[torch.Tensor, ...]:
    """An empty pool: (k_cache, v_cache, k_scale, v_scale)."""
    if head_dim not in HEAD_DIMS:
        raise RuntimeError(f"the int8 KV cache takes head_dim 64, 128 or 256, got {head_dim}")
    return (torch.zeros((pages, kv_heads, PAGE_TOKENS, head_dim), dtype=torch.int8, device=device),
            torch.zeros((pages, kv_heads, head_dim, PAGE_TOKENS), dtype=torch.int8, device=device),
            torch.zeros((pages, kv_heads), dtype=torch.float32, device=device),
            torch.zeros((pages, kv_heads), dtype=torch.float32, device=device))


def _strided(t: torch.Tensor) -> tuple[torch.Tensor, ctypes.Array]:
    """t [B, T, heads, D] with contiguous 16-byte aligned rows, copied only where it has none,
    and its first three strides."""
    st, sz = t.stride(), t.shape
    key = tuple(0 if sz[i] == 1 else st[i] for i in range(3))
    if st[3] != 1 or key[0] % 8 or key[1] % 8 or key[2] % 8 or t.data_ptr() % 16:
        t = t.clone(memory_format=torch.contiguous_format)
        key = t.stride()[:3]
    arr = _STRIDES.get(key)
    if arr is None:
        if len(_STRIDES) > 4096:
            _STRIDES.clear()
        arr = _STRIDES[key] = (ctypes.c_int64 * 3)(*key)
    return t, arr


def _check_cache(what, dev, k_cache, v_cache, k_scale, v_scale, table, lens, b, t, kvh, d):
    if d not in HEAD_DIMS:
        raise RuntimeError(f"{what}: head_dim must be 64, 128 or 256, got {d}")
    pages = k_cache.size(0) if k_cache.dim() else 0
    if k_cache.dtype != torch.int8 or k_cache.shape != (pages, kvh, PAGE_TOKENS, d):
        raise RuntimeError(f"{what}: k_cache must be int8 [pages, {kvh}, {PAGE_TOKENS}, {d}], got {k_cache.dtype} "
                           f"{tuple(k_cache.shape)}")
    if v_cache.dtype != torch.int8 or v_cache.shape != (pages, kvh, d, PAGE_TOKENS):
        raise RuntimeError(f"{what}: v_cache must be int8 [{pages}, {kvh}, {d}, {PAGE_TOKENS}], got {v_cache.dtype} "
                           f"{tuple(v_cache.shape)}")
    for name, s in (("k_scale", k_scale), ("v_scale", v_scale)):
        if s.dtype != torch.float32 or s.shape != (pages, kvh):
            raise RuntimeError(f"{what}: {name} must be float32 [{pages}, {kvh}], got {s.dtype} {tuple(s.shape)}")
    if table.dtype != torch.int32 or table.dim() != 2 or table.size(0) != b:
        raise RuntimeError(f"{what}: block_table must be int32 [{b}, pages of a sequence], got {table.dtype} "
                           f"{tuple(table.shape)}")
    if b > MAX_BATCH or t > MAX_TOKENS or table.size(1) > MAX_TOKENS:  # here: the library takes them as 32 bits
        raise RuntimeError(f"{what}: at most {MAX_BATCH} sequences, {MAX_TOKENS} tokens and {MAX_TOKENS} pages of a sequence, "
                           f"got {b}, {t} and {table.size(1)}")
    if lens.dtype != torch.int32 or lens.shape != (b,):
        raise RuntimeError(f"{what}: lens must be int32 [{b}], got {lens.dtype} {tuple(lens.shape)}")
    for c in (k_cache, v_cache, k_scale, v_scale, table, lens):
        if c.device != dev:
            raise RuntimeError(f"{what}: the cache, block_table and lens must be on {dev}, got {c.device}")
    if not (k_cache.is_contiguous() and v_cache.is_contiguous() and k_scale.is_contiguous() and v_scale.is_contiguous()):
        raise RuntimeError(f"{what}: the cache must be contiguous")
    if k_cache.data_ptr() % 16 or v_cache.data_ptr() % 16:
        raise RuntimeError(f"{what}: the cache must be 16-byte aligned")
    return pages


def _ints(what, name, t, b, dev):
    """An optional int32 [B] on the cache's device, contiguous."""
    if t is None:
        return None
    if t.dtype != torch.int32 or t.shape != (b,) or t.device != dev:
        raise RuntimeError(f"{what}: {name} must be int32 [{b}] on {dev}, got {t.dtype} {tuple(t.shape)} on {t.device}")
    return t.contiguous()


def _table(table: torch.Tensor) -> tuple[torch.Tensor, int]:
    if table.stride(1) != 1 and table.size(1) > 1:
        table = table.contiguous()
    return table, table.stride(0) if table.size(0) > 1 else table.size(1)


def _append_impl(k, v, k_cache, v_cache, k_scale, v_scale, block_table, lens, counts):
    what = "int8_kv_append"
    if not k.is_cuda:
        raise RuntimeError(f"{what} expects CUDA/HIP tensors")
    dev = k.device
    elem = ELEM.get(k.dtype)
    if elem is None or v.dtype != k.dtype:
        raise RuntimeError(f"{what} takes float16 or bfloat16 keys and values of one type, got {k.dtype} and {v.dtype}")
    if k.dim() != 4 or v.shape != k.shape or v.device != dev:
        raise RuntimeError(f"{what} expects k and v [B, T, KVH, D] on one device, got {tuple(k.shape)} and {tuple(v.shape)}")
    b, t, kvh, d = k.shape
    pages = _check_cache(what, dev, k_cache, v_cache, k_scale, v_scale, block_table, lens, b, t, kvh, d)
    counts = _ints(what, "counts", counts, b, dev)
    if b == 0 or t == 0:
        return
    table, stride = _table(block_table)
    lens = lens.contiguous()
    k, ks = _strided(k)
    v, vs = _strided(v)
    lib = _ext._lib if _ext._lib is not None else load_int4_gemm()
    with _on_device(dev):
        _check(lib.pi05w4a4_int8_kv_append(k.data_ptr(), ks, v.data_ptr(), vs, elem, b, t, kvh, d, k_cache.data_ptr(),
                                           v_cache.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(), pages,
                                           table.data_ptr(), stride, table.size(1), lens.data_ptr(), _ptr(counts),
                                           _stream(dev)), "pi05w4a4_int8_kv_append")


def _attention_impl(q, k_cache, v_cache, k_scale, v_scale, block_table, lens, scaling, causal, q_lens, return_lse):
    what = "int8_kv_attention"
    if not q.is_cuda:
        raise RuntimeError(f"{what} expects CUDA/HIP tensors")
    dev = q.device
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
    pages = _check_cache(what, dev, k_cache, v_cache, k_scale, v_scale, block_table, lens, b, t, kvh, d)
    q_lens = _ints(what, "q_lens", q_lens, b, dev)
    out = torch.empty_like(q, memory_format=torch.contiguous_format)
    lse = torch.empty((b, t, h), dtype=torch.float32, device=dev) if return_lse else None
    if b == 0 or t == 0:
        return out, lse
    table, stride = _table(block_table)
    lens = lens.contiguous()
    q, qs = _strided(q)
    tp = table.size(1)
    lib = _ext._lib if _ext._lib is not None else load_int4_gemm()
    with _on_device(dev):
        key = (dev.index, b, t, h, kvh, d, tp)
        need = _ATTN_WS.get(key)
        if need is None:
            if len(_ATTN_WS) > 4096:
                _ATTN_WS.clear()
            need = _ATTN_WS[key] = int(lib.pi05w4a4_int8_kv_attention_workspace_bytes(b, t, h, kvh, d, tp))
        ws = _workspace(dev, need) if need else None
        _check(lib.pi05w4a4_int8_kv_attention(q.data_ptr(), qs, elem, b, t, h, kvh, d, k_cache.data_ptr(),
                                              v_cache.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(), pages,
                                              table.data_ptr(), stride, tp, lens.data_ptr(), _ptr(q_lens), scaling,
                                              1 if causal else 0, out.data_ptr(), _ptr(lse), _ptr(ws), need,
                                              _stream(dev)), "pi05w4a4_int8_kv_attention")
    return out, lse


# ----------------------------------------------------------------------------- custom ops
@torch.library.custom_op("pi05_w4a4::int8_kv_append", mutates_args=("k_cache", "v_cache", "k_scale", "v_scale"))
def _append_op(k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, k_scale: torch.Tensor,
               v_scale: torch.Tensor, block_table: torch.Tensor, lens: torch.Tensor,
               counts: torch.Tensor | None) -> None:
    _refuse_tangents(k, v, k_scale, v_scale)
    _append_impl(k, v, k_cache, v_cache, k_scale, v_scale, block_table, lens, counts)


@_append_op.register_fake
def _append_fake(k, v, k_cache, v_cache, k_scale, v_scale, block_table, lens, counts):
    return None


@torch.library.custom_op("pi05_w4a4::int8_kv_attention", mutates_args=())
def _attention_op(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, k_scale: torch.Tensor,
                  v_scale: torch.Tensor, block_table: torch.Tensor, lens: torch.Tensor, scaling: float, causal: bool,
                  q_lens: torch.Tensor | None, return_lse: bool) -> tuple[torch.Tensor, torch.Tensor]:
    _refuse_tangents(q, k_scale, v_scale)
    out, lse = _attention_impl(q, k_cache, v_cache, k_scale, v_scale, block_table, lens, scaling, causal, q_lens,
                               return_lse)
    return out, lse if lse is not None else out.new_empty((0,), dtype=torch.float32)


@_attention_op.register_fake
def _attention_fake(q, k_cache, v_cache, k_scale, v_scale, block_table, lens, scaling, causal, q_lens, return_lse):
    return q.new_empty(q.shape), q.new_empty(q.shape[:-1] if return_lse else (0,), dtype=torch.float32)


# ----------------------------------------------------------------------------- public functions
def int8_kv_append(k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                   k_scale: torch.Tensor, v_scale: torch.Tensor, block_table: torch.Tensor, lens: torch.Tensor,
                   counts: torch.Tensor | None = None) -> None:
    """Write k and v [B, T, KVH, D] (fp16 or bf16, any strides) behind each sequence's
    ``lens`` [B] cached tokens, the first ``counts`` [B] of them (None: all T); the rest of
    a padded batch is not read.  Changes the cache in place and leaves ``lens`` as it is.

    A page's scale is max|value| / 127 + 1e-12 over its tokens.  Where it grows, the page's
    earlier codes are rounded to it; a page whose first token is new is written whole, with
    zeros behind the last token.  No other page is touched.  A NaN or infinity makes its
    page's scale NaN.  Tokens past the table, or whose table entry names no page, are
    dropped.  A call may write a page from one place only: full pages can be shared between
    sequences, and stand in a table twice, a page that still fills cannot."""
    if _direct(k, v, k_cache, v_cache, k_scale, v_scale, block_table, lens, counts):
        _append_impl(k, v, k_cache, v_cache, k_scale, v_scale, block_table, lens, counts)
        return _changed((k_cache, v_cache, k_scale, v_scale))
    return torch.ops.pi05_w4a4.int8_kv_append(k, v, k_cache, v_cache, k_scale, v_scale, block_table, lens, counts)


def int8_kv_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, k_scale: torch.Tensor,
                      v_scale: torch.Tensor, block_table: torch.Tensor, lens: torch.Tensor, scaling: float,
                      causal: bool = True, q_lens: torch.Tensor | None = None, return_lse: bool = False):
    """softmax(scaling q K^T) V of q [B, T, H, D] (fp16 or bf16, RoPE applied, any strides)
    over the cache: [B, T, H, D] in q's type.  H is a multiple of KVH; query head h reads KV
    head h // (H / KVH).  The work is planned for the table's width: pass a table held at
    capacity as ``block_table[:, :n]``, n the pages of the longest sequence.  Entries that name
    no page hide their 64 tokens.

    The queries are the last T tokens (``q_lens`` [B]: the last q_lens[b], the rows behind
    them padding) of ``lens`` [B] cached ones, whose keys the cache holds already.  When
    ``causal``, query i sees the first lens - q_len + i + 1 tokens, else all of them.  A length
    past the table (64 tokens an entry) counts as the table's, for the place of the queries
    too: where an append dropped tokens, ``q_lens`` without their queries gives the others what
    they see.  A query that sees no token, a padding row among them, gets zeros.  With ``return_lse``, also the
    natural log of the sum of exp(scaling q k), fp32 [B, T, H] (-inf where none is seen), with
    which attention over further keys can be joined."""
    if _direct(q, k_cache, v_cache, k_scale, v_scale, block_table, lens, q_lens):
        out, lse = _attention_impl(q, k_cache, v_cache, k_scale, v_scale, block_table, lens, float(scaling),
                                   bool(causal), q_lens, bool(return_lse))
    else:
        out, lse = torch.ops.pi05_w4a4.int8_kv_attention(q, k_cache, v_cache, k_scale, v_scale, block_table, lens,
                                                         float(scaling), bool(causal), q_lens, bool(return_lse))
    return (out, lse) if return_lse else out
