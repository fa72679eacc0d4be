"""Drafted tokens of a serving step for torch device tensors, over the C ABI of
include/ifx_drafts.h: trees of drafts in the attention over the paged cache,
which of them the target's probabilities accept, and what the cache keeps.

    # per step: request b brings the nodes of a tree, its last token the root;
    # parents[t] is the node before the one of row t, -1 of a root
    p = attention.plan_batch(ctx_len, new_len, table, free, free_count, 64, T)
    t = drafts.plan_tree(parents, p.cu_q, p.kv_len)
    # per layer, with the caches and the workspace of `attention`
    q = attention.rope_append(q, k, v, t.positions, p.slots, k_cache, v_cache, inv_freq)
    o = drafts.tree_attention(q, k_cache, v_cache, table, p.cu_q, p.kv_len, t.masks, max_q, max_kv,
                              workspace=ws)
    # behind the LM head: the target's probabilities [T, vocab]
    r = drafts.verify(tokens, p.cu_q, probs, accept_u, sample_u, max_q, parents=parents, workspace=ws)
    for k_cache, v_cache in layers:
        drafts.keep_path((k_cache, v_cache), table, p.cu_q, p.kv_len, r.path, r.accepted, max_q)
    kept = drafts.plan_kept(p.cu_q, p.kv_len, r.accepted, table, free, p.free_left, 64)
    # the next step's ctx_len and free_count are kept.ctx_len and kept.free_left

A request has at most MAX_NODES nodes.  The 8-bit cache's attention takes the
same masks (attention_q8.paged_attention), and keep_path an attention_q8.Q8Cache.
What `attention` says of types, streams, captured graphs and errors holds here.
"""
from collections import namedtuple

import torch

from . import _lib
from .attention import _DTYPES, _caches, _count, _device, _i32, _launch, _new, _on, _out, _rows

MAX_NODES = 64
# bits of KeptPlan.status
NO_SPACE = 1

TreePlan = namedtuple("TreePlan", "positions masks")
Verified = namedtuple("Verified", "accepted path emitted")
KeptPlan = namedtuple("KeptPlan", "ctx_len free_left status")


def _made(shape, dtype, like, stream):
    """attention's _new, sooner where the output is the current stream's."""
    return like.new_empty(shape, dtype=dtype) if stream is None else _new(shape, dtype, like, stream)


def _masks(t, n, device):
    if t.dtype is not torch.int64:
        raise TypeError("masks must be int64")
    if t.numel() < n or not t.is_contiguous():
        raise ValueError(f"masks must be contiguous with at least {n} values")
    return _on(t, "masks", device).data_ptr()


def _all_on(device, *tensors):
    for t in tensors:
        if t.get_device() != device:
            raise ValueError(f"all tensors of a call must be on cuda:{device}")


def _q8_caches(c):
    """(pages, kv heads, page size, head size) of an attention_q8.Q8Cache."""
    k, v, s = c
    if k.dtype is not torch.int8 or v.dtype is not torch.int8 or s.dtype is not torch.bfloat16:
        raise TypeError("an 8-bit cache has int8 codes and bfloat16 scales")
    shape = k.shape
    if len(shape) == 5:
        n, h, d16, p, e = shape
        if e == 16 and v.shape == (n, h, p // 16, d16 * 16, 16) and s.shape == (n, h, p, 2):
            if not (k.is_contiguous() and v.is_contiguous() and s.is_contiguous()):
                raise ValueError("the cache must be contiguous")
            return n, h, p, d16 * 16
    raise ValueError("the cache must be as kv_cache makes it: [pages, heads, D / 16, page, 16], "
                     "[pages, heads, page / 16, D, 16] and [pages, heads, page, 2]")


def _f32(t, name, n, device):
    if t.dtype is not torch.float32:
        raise TypeError(f"{name} must be float32")
    if t.numel() < n or not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous with at least {n} values")
    return _on(t, name, device).data_ptr()


def _table(t, B):
    if t.dim() != 2 or t.shape[0] != B:
        raise ValueError("block_table must be [B, pages]")
    return t.shape[1]


def plan_tree(parents, cu_q, kv_len, out=None, stream=None):
    """Positions and masks of the nodes of a batch's trees (ifx_plan_tree).
    parents [T]: per row its parent's row in the request, an earlier one; any
    other number (-1): none.  Returns a TreePlan (`out`: one of an earlier call
    to write into): positions [T] int32, the cached tokens and the node's depth,
    and masks [T] int64, bit j: node j is the node itself or on its way to the
    root.  Rows past a request's first MAX_NODES and behind cu_q[B]: 0."""
    dev, T, B = _device(parents, "parents"), parents.numel(), kv_len.numel()
    if out is None:
        out = TreePlan(_made((T,), torch.int32, parents, stream), _made((T,), torch.int64, parents, stream))
    _launch(_lib.load().ifx_plan_tree, "ifx_plan_tree", dev, stream, _i32(parents, "parents", T, dev),
            _i32(cu_q, "cu_q", B + 1, dev), _i32(kv_len, "kv_len", B, dev), B, T,
            _i32(out.positions, "positions", T, dev), _masks(out.masks, T, dev))
    return out


def tree_attention(q, k_cache, v_cache, block_table, cu_q, kv_len, masks, max_q, max_kv, scale=None,
                   out=None, out_dtype=None, workspace=None, stream=None):
    """attention.paged_attention of drafted trees (ifx_attn_tree): row i of a
    request of n new tokens sees the tokens before those, and the new ones j
    whose bit is set in masks[row], int64 [T] as plan_tree makes them.
    max_q <= MAX_NODES."""
    n, Hkv, P, D = _caches(k_cache, v_cache)
    dev = _device(q, "q")
    if q.dim() != 3:
        raise ValueError("q must be [T, Hq, D]")
    if q.dtype is not k_cache.dtype:
        raise TypeError("q must have the caches' type")
    T, Hq = q.shape[0], q.shape[1]
    B = kv_len.numel()
    W = _table(block_table, B)
    out = _out(q, out, out_dtype, stream)
    _all_on(dev, k_cache, v_cache, out)
    qp, qs = _rows(q, "q", T, Hq, D)
    op, os = _rows(out, "out", T, Hq, D)
    wp, wn = _workspace(workspace, dev)
    _launch(_lib.load().ifx_attn_tree, "ifx_attn_tree", dev, stream, qp, qs, _DTYPES[q.dtype],
            k_cache.data_ptr(), v_cache.data_ptr(), n, P,
            _i32(block_table, "block_table", B * W, dev), W, _i32(cu_q, "cu_q", B + 1, dev),
            _i32(kv_len, "kv_len", B, dev), _masks(masks, T, dev), B, T, Hq, Hkv, D,
            _count(max_q, "max_q"), _count(max_kv, "max_kv"), D ** -0.5 if scale is None else scale,
            op, os, _DTYPES[out.dtype], wp, wn)
    return out


def tree_workspace_bytes(B, T, Hq, Hkv, head_dim, max_q, max_kv):
    """Bytes of workspace that tree_attention needs for this shape (0: none;
    attention.WORKSPACE_BYTES is enough for all)."""
    return int(_lib.load().ifx_attn_tree_workspace_bytes(
        _count(B, "B"), _count(T, "T"), _count(Hq, "Hq"), _count(Hkv, "Hkv"),
        _count(head_dim, "head_dim"), _count(max_q, "max_q"), _count(max_kv, "max_kv")))


def _workspace(t, device):
    if t is None:
        return None, 0
    if not t.is_contiguous():
        raise ValueError("workspace must be contiguous")
    return _on(t, "workspace", device).data_ptr(), t.nbytes


def _probs(t, name, T, dtype, device):
    """Pointer and row stride of probabilities [T, V]."""
    if t.dim() != 2 or t.shape[0] != T:
        raise ValueError(f"{name} must be [{T}, vocab]")
    if t.dtype not in _DTYPES or t.dtype is not dtype:
        raise TypeError("probabilities must be float32, float16 or bfloat16, all the same")
    V = t.shape[1]
    if T and V > 1 and t.stride(1) != 1:
        raise ValueError(f"{name}: a row's values must lie one after the other")
    return _on(t, name, device).data_ptr(), t.stride(0) if T > 1 else V


def verify_workspace_bytes(B, vocab):
    """Bytes of workspace that verify needs (attention.WORKSPACE_BYTES is enough)."""
    return int(_lib.load().ifx_verify_workspace_bytes(_count(B, "B"), _count(vocab, "vocab")))


def verify(tokens, cu_q, target_probs, accept_u, sample_u, max_q, parents=None, draft_probs=None,
           out=None, workspace=None, stream=None):
    """Which drafted nodes the target accepts and the token behind them
    (ifx_verify).  tokens [T]: the nodes' tokens, rows of the requests as cu_q
    [B + 1] has them; target_probs [T, vocab]: row t the target's probabilities
    behind node t; accept_u [T] and sample_u [B]: float32 in [0, 1).  max_q
    bounds a request's rows, MAX_NODES at most.

    Without draft_probs the drafts are choices: from node i to its first child
    (parents [T] as in plan_tree, a chain if None) with accept_u[i] below the
    probabilities of its token and its earlier siblings' together.  With
    draft_probs [T, vocab] they are a chain that was drawn from it: on to node
    i + 1 with token x where accept_u[i] * draft_probs[i, x] < target_probs[i, x].
    The next token is drawn with sample_u from what is left of the target's
    probabilities at the last node.

    Returns Verified of int32 tensors (`out`: one of an earlier call to write
    into): accepted [B] drafts (-1: the request has no rows); path [T], the
    nodes walked from the root on, and emitted [T], the accepted drafts' tokens
    and the one drawn, both request by request and filled with -1."""
    dev, T, B = _device(tokens, "tokens"), tokens.numel(), cu_q.numel() - 1
    if parents is not None and draft_probs is not None:
        raise ValueError("drafts with probabilities are a chain: parents must be None")
    tp, ts = _probs(target_probs, "target_probs", T, target_probs.dtype, dev)
    V = target_probs.shape[1]
    dp, ds = None, 0
    if draft_probs is not None:
        if draft_probs.shape != target_probs.shape:
            raise ValueError("draft_probs must have the shape of target_probs")
        dp, ds = _probs(draft_probs, "draft_probs", T, target_probs.dtype, dev)
    if B < 1:
        raise ValueError("cu_q must have a value for each request and one more")
    if workspace is None:
        raise ValueError("verify needs a workspace")
    wp, wn = _workspace(workspace, dev)
    if out is None:
        out = Verified(*_made(B + 2 * T, torch.int32, tokens, stream).split_with_sizes((B, T, T)))
    _launch(_lib.load().ifx_verify, "ifx_verify", dev, stream, _i32(tokens, "tokens", T, dev),
            None if parents is None else _i32(parents, "parents", T, dev),
            _i32(cu_q, "cu_q", B + 1, dev), B, T, _count(max_q, "max_q"), tp, ts, dp, ds,
            _DTYPES[target_probs.dtype], V, _f32(accept_u, "accept_u", T, dev),
            _f32(sample_u, "sample_u", B, dev), _i32(out.accepted, "accepted", B, dev),
            _i32(out.path, "path", T, dev), _i32(out.emitted, "emitted", T, dev), wp, wn)
    return out


def keep_path(cache, block_table, cu_q, kv_len, path, accepted, max_q, stream=None):
    """Moves the K and V of the accepted nodes behind the tokens that one
    layer's cache held before the step (ifx_keep_path); cache: (k_cache,
    v_cache) of attention.kv_cache or an attention_q8.Q8Cache; path [T] and
    accepted [B] as verify returns them."""
    if len(cache) == 3:
        n, Hkv, P, D = _q8_caches(cache)
    else:
        n, Hkv, P, D = _caches(*cache)
    dev, B, T = _device(cache[0], "k_cache"), kv_len.numel(), path.numel()
    _all_on(dev, *cache)
    W = _table(block_table, B)
    _launch(_lib.load().ifx_keep_path, "ifx_keep_path", dev, stream, cache[0].data_ptr(),
            cache[1].data_ptr(), cache[2].data_ptr() if len(cache) == 3 else None,
            cache[0].element_size(), n, P, Hkv, D, _i32(block_table, "block_table", B * W, dev), W,
            _i32(cu_q, "cu_q", B + 1, dev), _i32(kv_len, "kv_len", B, dev), _i32(path, "path", T, dev),
            _i32(accepted, "accepted", B, dev), B, T, _count(max_q, "max_q"))


def plan_kept(cu_q, kv_len, accepted, block_table, free_pages, free_count, page_size, out=None,
              stream=None):
    """The lengths that a batch goes on with, and the pages that its rejected
    drafts took (ifx_plan_kept): these are put back behind
    free_pages[:free_count[0]], free_count being plan_batch's free_left.
    Returns a KeptPlan of int32 tensors (`out`: one of an earlier call to write
    into): ctx_len [B], free_left [1], status [1] (0, or NO_SPACE: then no page
    is given back)."""
    dev, B = _device(kv_len, "kv_len"), kv_len.numel()
    W = _table(block_table, B)
    if out is None:
        out = KeptPlan(*_made(B + 2, torch.int32, kv_len, stream).split_with_sizes((B, 1, 1)))
    _launch(_lib.load().ifx_plan_kept, "ifx_plan_kept", dev, stream, _i32(cu_q, "cu_q", B + 1, dev),
            _i32(kv_len, "kv_len", B, dev), _i32(accepted, "accepted", B, dev),
            _i32(block_table, "block_table", B * W, dev), W, _i32(free_pages, "free_pages", 0, dev),
            free_pages.numel(), _i32(free_count, "free_count", 1, dev), _count(page_size, "page_size"),
            B, _i32(out.ctx_len, "ctx_len", B, dev), _i32(out.free_left, "free_left", 1, dev),
            _i32(out.status, "status", 1, dev))
    return out
