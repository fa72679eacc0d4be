"""The 8-bit paged cache for torch device tensors, over the C ABI of
include/ifx_attention_q8.h: K and V quantised as they are written, the attention
over them, and tokens read back.  Half the memory of attention's cache, and half
the bytes of a decode step.

    cache = attention_q8.kv_cache(pages, kv_heads, head_dim)         # per layer
    ws = attention.workspace()                                       # per stream

    p = attention.plan_batch(ctx_len, new_len, table, free, free_count, 64, T)
    q = attention_q8.rope_append(q, k, v, p.positions, p.slots, cache, inv_freq)
    o = attention_q8.paged_attention(q, cache, table, p.cu_q, p.kv_len, max_q, max_kv,
                                     workspace=ws, out_dtype=torch.float16)

A value is an int8 code times a bfloat16 scale, one for K and one for V of each
token and head.  Requests may bring trees of drafts (`drafts`): masks of
drafts.plan_tree, drafts.keep_path.  What `attention` says of types, streams,
captured graphs and errors holds here.
"""
from collections import namedtuple

import torch

from . import _lib
from .attention import _DTYPES, _ELEMS, PAGE_SIZES, _count, _device, _i32, _launch, _on, _out, _rows
from .drafts import _all_on, _made, _masks, _q8_caches, _table, _workspace

Q8Cache = namedtuple("Q8Cache", "k v scales")


def kv_cache(num_pages, kv_heads, head_dim, page_size=64, device="cuda"):
    """One layer's 8-bit paged cache, zeroed: a Q8Cache of codes and scales in
    the layout of include/ifx_attention_q8.h."""
    if page_size not in PAGE_SIZES:
        raise ValueError(f"page_size must be one of {PAGE_SIZES}")
    if head_dim % 32 or not 0 < head_dim <= 256:
        raise ValueError("head_dim must be a multiple of 32 up to 256")
    return Q8Cache(
        torch.zeros(num_pages, kv_heads, head_dim // 16, page_size, 16, dtype=torch.int8, device=device),
        torch.zeros(num_pages, kv_heads, page_size // 16, head_dim, 16, dtype=torch.int8, device=device),
        torch.zeros(num_pages, kv_heads, page_size, 2, dtype=torch.bfloat16, device=device))


def rope_append(q, k, v, positions, slots, cache, inv_freq=None, interleaved=False, q_out=None,
                q_dtype=None, stream=None):
    """attention.rope_append into an 8-bit cache (ifx_rope_append_q8): rotates q
    [T, Hq, D] and k [T, Hkv, D], writes k and v as codes and scales at `slots`,
    and returns the rotated q in q_dtype (float16 if None, or q_out's type)."""
    n, Hkv, P, D = _q8_caches(cache)
    dev = _device(cache.k, "cache.k")
    if q.dim() != 3:
        raise ValueError("q must be [T, Hq, D]")
    T, Hq = q.shape[0], q.shape[1]
    src = _DTYPES.get(q.dtype)
    if src is None or k.dtype is not q.dtype or v.dtype is not q.dtype:
        raise TypeError("q, k and v must be float32, float16 or bfloat16, all the same")
    want = q_dtype or (torch.float16 if q_out is None else q_out.dtype)
    if want not in _ELEMS or (q_out is not None and q_out.dtype is not want):
        raise TypeError("q_out must be float16 or bfloat16, and of q_dtype if that is given")
    rot, freq = 0, None
    if inv_freq is not None:
        if inv_freq.dtype is not torch.float64 or not inv_freq.is_contiguous():
            raise TypeError("inv_freq must be contiguous float64")
        rot, freq = 2 * inv_freq.numel(), _on(inv_freq, "inv_freq", dev).data_ptr()
    if q_out is None:
        q_out = _made((T, Hq, D), want, cache.k, stream)
    _all_on(dev, q, k, v, cache.v, cache.scales, q_out)
    qp, qs = _rows(q, "q", T, Hq, D)
    kp, ks = _rows(k, "k", T, Hkv, D)
    vp, vs = _rows(v, "v", T, Hkv, D)
    op, os = _rows(q_out, "q_out", T, Hq, D)
    _launch(_lib.load().ifx_rope_append_q8, "ifx_rope_append_q8", dev, stream, qp, qs, kp, ks, vp, vs,
            src, _i32(positions, "positions", T, dev), _i32(slots, "slots", T, dev), freq, rot,
            1 if interleaved else 0, T, Hq, Hkv, D, op, os, _DTYPES[want], cache.k.data_ptr(),
            cache.v.data_ptr(), cache.scales.data_ptr(), n, P)
    return q_out


def read_rows(cache, slots, dtype=torch.float16, k_out=None, v_out=None, stream=None):
    """The values that the tokens at `slots` [N] hold (ifx_read_rows_q8): k and v
    [N, Hkv, D] in `dtype` (fp32, fp16 or bf16; that of k_out and v_out where
    they are given), 0 for a slot outside the cache."""
    n, Hkv, P, D = _q8_caches(cache)
    dev, N = _device(cache.k, "cache.k"), slots.numel()
    k_out = _made((N, Hkv, D), dtype, cache.k, stream) if k_out is None else k_out
    v_out = _made((N, Hkv, D), k_out.dtype, cache.k, stream) if v_out is None else v_out
    if k_out.dtype not in _DTYPES or v_out.dtype is not k_out.dtype:
        raise TypeError("k_out and v_out must be float32, float16 or bfloat16, both the same")
    _all_on(dev, cache.v, cache.scales, k_out, v_out)
    kp, ks = _rows(k_out, "k_out", N, Hkv, D)
    vp, vs = _rows(v_out, "v_out", N, Hkv, D)
    _launch(_lib.load().ifx_read_rows_q8, "ifx_read_rows_q8", dev, stream, cache.k.data_ptr(),
            cache.v.data_ptr(), cache.scales.data_ptr(), n, P, _i32(slots, "slots", N, dev), N, Hkv, D,
            kp, ks, vp, vs, _DTYPES[k_out.dtype])
    return k_out, v_out


def paged_workspace_bytes(B, T, Hq, Hkv, head_dim, max_q, max_kv):
    """Bytes of workspace that paged_attention needs for this shape (0: none;
    attention.WORKSPACE_BYTES is enough for all)."""
    return int(_lib.load().ifx_attn_paged_q8_workspace_bytes(
        _count(B, "B"), _count(T, "T"), _count(Hq, "Hq"), _count(Hkv, "Hkv"),
        _count(head_dim, "head_dim"), _count(max_q, "max_q"), _count(max_kv, "max_kv")))


def paged_attention(q, cache, block_table, cu_q, kv_len, max_q, max_kv, scale=None, window=0, masks=None,
                    out=None, out_dtype=None, workspace=None, stream=None):
    """attention.paged_attention over an 8-bit cache (ifx_attn_paged_q8), q
    float16 or bfloat16.  masks: of drafted trees, as drafts.tree_attention's
    (window 0 then).  workspace: attention.workspace, or paged_workspace_bytes of it."""
    n, Hkv, P, D = _q8_caches(cache)
    dev = _device(q, "q")
    if q.dim() != 3:
        raise ValueError("q must be [T, Hq, D]")
    if q.dtype not in _ELEMS:
        raise TypeError("q must be float16 or bfloat16")
    T, Hq = q.shape[0], q.shape[1]
    B = kv_len.numel()
    W = _table(block_table, B)
    out = _out(q, out, out_dtype, stream)
    _all_on(dev, cache.k, cache.v, cache.scales, out)
    qp, qs = _rows(q, "q", T, Hq, D)
    op, os = _rows(out, "out", T, Hq, D)
    wp, wn = _workspace(workspace, dev)
    _launch(_lib.load().ifx_attn_paged_q8, "ifx_attn_paged_q8", dev, stream, qp, qs, _DTYPES[q.dtype],
            cache.k.data_ptr(), cache.v.data_ptr(), cache.scales.data_ptr(), n, P,
            _i32(block_table, "block_table", B * W, dev), W, _i32(cu_q, "cu_q", B + 1, dev),
            _i32(kv_len, "kv_len", B, dev), None if masks is None else _masks(masks, T, dev), B, T, Hq,
            Hkv, D, _count(max_q, "max_q"), _count(max_kv, "max_kv"), D ** -0.5 if scale is None else scale,
            _count(window, "window"), op, os, _DTYPES[out.dtype], wp, wn)
    return out
