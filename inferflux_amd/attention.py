"""The attention of a serving step for torch device tensors, over the C ABI of
include/ifx_attention.h: what lies between a layer's Q/K/V projections and its
O projection (`ops`).

    k_cache, v_cache = attention.kv_cache(pages, kv_heads, head_dim)   # per layer
    ws = attention.workspace()                                         # per stream

    # per step: B requests, new_len[b] new tokens behind ctx_len[b] cached ones
    p = attention.plan_batch(ctx_len, new_len, table, free, free_count, 64, T)
    # per layer: the projections' rows q [T, Hq, D], k and v [T, Hkv, D]
    q = attention.rope_append(q, k, v, p.positions, p.slots, k_cache, v_cache, inv_freq)
    o = attention.paged_attention(q, k_cache, v_cache, table, p.cu_q, p.kv_len,
                                  max_q, max_kv, workspace=ws, out_dtype=torch.float16)

Whole prompts that no cache is kept for (scoring, embedding) go through
prompt_attention instead.  Integers are int32, caches and rows of Q fp16 or
bf16.  Nothing here synchronises the host, and with outputs given nothing
allocates, so every call can be captured into a graph.  Calls run on the
current stream of the tensors' device, or on `stream`, one of that device; what
they return there is read elsewhere only after a wait for `stream`.
Errors are those of `ops`: NotHandled, HipError, ValueError, TypeError.
"""
from collections import namedtuple

import torch

from . import _lib
from .ops import _check

MAX_BATCH = 4096
WORKSPACE_BYTES = 64 << 20  # IFX_ATTN_WORKSPACE_BYTES: enough for every call
PAGE_SIZES = (16, 32, 64, 128, 256)
HEAD_DIMS = (64, 96, 128, 256)
# bits of BatchPlan.status
NO_PAGES, NARROW, NO_ROOM, BAD_LENGTH = 1, 2, 4, 8

_DTYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
_ELEMS = (torch.float16, torch.bfloat16)

BatchPlan = namedtuple("BatchPlan", "cu_q kv_len positions slots free_left status")


def _launch(fn, what, device, stream, *args):
    """Calls a C entry point on `stream` or the current one of device number
    `device`, which is made the current device for the call if it is not."""
    if stream is None:
        raw = torch._C._cuda_getCurrentRawStream(device)
    elif stream.device_index != device:
        raise ValueError(f"the stream is of cuda:{stream.device_index}, the tensors of cuda:{device}")
    else:
        raw = stream.cuda_stream
    if device == torch._C._cuda_getDevice():
        rc = fn(*args, raw)
    else:
        with torch.cuda.device(device):
            rc = fn(*args, raw)
    if rc:
        _check(rc, what)


def _device(t, name):
    """Number of the GPU that t is on; the other tensors of a call are held to it."""
    if not t.is_cuda:
        raise ValueError(f"{name} must be a device tensor")
    return t.get_device()


def _new(shape, dtype, like, stream):
    """An output of a call.  On a given stream it is that stream's own memory:
    the current one's may be a block just freed there, with work on it still
    pending that `stream` does not wait for.  The caller goes on with it on the
    current stream, so the allocator is told of that one."""
    if stream is None:
        return torch.empty(shape, dtype=dtype, device=like.device)
    user = torch.cuda.current_stream(like.device)
    with torch.cuda.stream(stream):
        t = torch.empty(shape, dtype=dtype, device=like.device)
    t.record_stream(user)
    return t


def _count(v, name):
    """A size or length as the C entries take it: ctypes would drop the bits
    that do not fit."""
    if not 0 <= v < 1 << 31:
        raise ValueError(f"{name} must be from 0 to 2^31 - 1, got {v}")
    return v


def _on(t, name, device):
    if t.get_device() != device:
        raise ValueError(f"{name} must be on cuda:{device}")
    return t


def _i32(t, name, n, device):
    if t.dtype is not torch.int32:
        raise TypeError(f"{name} must be int32")
    if t.get_device() != device:
        raise ValueError(f"{name} must be on cuda:{device}")
    if t.numel() < n or not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous with at least {n} values")
    return t.data_ptr()


def _rows(t, name, T, H, D):
    """Pointer and row stride of rows [T, H, D]: heads of D values one after
    the other, rows any distance apart."""
    if tuple(t.shape) != (T, H, D):
        raise ValueError(f"{name} must be [{T}, {H}, {D}], got {list(t.shape)}")
    row, head, one = t.stride()
    if T <= 1:
        row = H * D
    if T and ((one != 1 and D > 1) or (head != D and H > 1)):
        raise ValueError(f"{name}: a row's heads must lie one after the other")
    return t.data_ptr(), row


def _caches(k_cache, v_cache):
    """(pages, kv heads, page size, head size) of a layer's caches."""
    if k_cache.dtype not in _ELEMS or v_cache.dtype is not k_cache.dtype:
        raise TypeError("the caches must be float16 or bfloat16, both the same")
    if k_cache.dim() == 5 and v_cache.dim() == 5:
        n, h, d8, p, e = k_cache.shape
        if e == 8 and tuple(v_cache.shape) == (n, h, p // 8, d8 * 8, 8):
            if not k_cache.is_contiguous() or not v_cache.is_contiguous():
                raise ValueError("the caches must be contiguous")
            return n, h, p, d8 * 8
    raise ValueError("the caches must be as kv_cache makes them: [pages, heads, D / 8, page, 8] "
                     "and [pages, heads, page / 8, D, 8]")


def kv_cache(num_pages, kv_heads, head_dim, page_size=64, dtype=torch.float16, device="cuda"):
    """One layer's paged cache (K, V), zeroed: num_pages pages of page_size
    tokens, in the layout of include/ifx_attention.h."""
    if page_size not in PAGE_SIZES:
        raise ValueError(f"page_size must be one of {PAGE_SIZES}")
    if head_dim % 8 or dtype not in _ELEMS:
        raise ValueError("head_dim must be a multiple of 8, dtype float16 or bfloat16")
    k = torch.zeros(num_pages, kv_heads, head_dim // 8, page_size, 8, dtype=dtype, device=device)
    v = torch.zeros(num_pages, kv_heads, page_size // 8, head_dim, 8, dtype=dtype, device=device)
    return k, v


def workspace(device="cuda"):
    """A workspace for paged_attention's split sums that is large enough for
    any call.  One per stream: calls that share one must not overlap."""
    return torch.zeros(WORKSPACE_BYTES, dtype=torch.uint8, device=device)


def plan_batch(ctx_len, new_len, block_table, free_pages, free_count, page_size, max_tokens,
               out=None, stream=None):
    """Pages, slots, positions and row offsets of one step, on the device
    (ifx_plan_batch).  ctx_len, new_len [B]; block_table [B, W], updated in
    place; free_pages: a stack of free page numbers of which the first
    free_count[0] are valid, taken from the end.  Returns a BatchPlan of int32
    tensors (`out`: one of an earlier call to write into):

      cu_q [B + 1], kv_len [B], positions and slots [max_tokens] (behind the
      last token: 0 and -1), free_left [1], status [1] (0, or a sum of
      NO_PAGES, NARROW, NO_ROOM, BAD_LENGTH: then nothing is taken, cu_q is 0
      and every slot -1)."""
    dev, B = _device(ctx_len, "ctx_len"), ctx_len.numel()
    page_size, max_tokens = _count(page_size, "page_size"), _count(max_tokens, "max_tokens")
    if block_table.dim() != 2 or block_table.shape[0] != B:
        raise ValueError("block_table must be [B, pages]")
    if out is None:
        n = (B + 1, B, max_tokens, max_tokens, 1, 1)
        out = BatchPlan(*_new(sum(n), torch.int32, ctx_len, stream).split(n))
    W = block_table.shape[1]
    _launch(_lib.load().ifx_plan_batch, "ifx_plan_batch", dev, stream,
            _i32(ctx_len, "ctx_len", B, dev), _i32(new_len, "new_len", B, dev),
            _i32(block_table, "block_table", B * W, dev), W,
            _i32(free_pages, "free_pages", 0, dev), free_pages.numel(),
            _i32(free_count, "free_count", 1, dev), page_size, B, max_tokens,
            _i32(out.cu_q, "cu_q", B + 1, dev), _i32(out.kv_len, "kv_len", B, dev),
            _i32(out.positions, "positions", max_tokens, dev),
            _i32(out.slots, "slots", max_tokens, dev),
            _i32(out.free_left, "free_left", 1, dev), _i32(out.status, "status", 1, dev))
    return out


def rope_append(q, k, v, positions, slots, k_cache, v_cache, inv_freq=None, interleaved=False,
                q_out=None, stream=None):
    """Rotates q [T, Hq, D] and k [T, Hkv, D] by positions * inv_freq and writes
    k and v into the caches at `slots` (ifx_rope_append); returns the rotated
    q in the caches' type.  q, k and v: fp32, fp16 or bf16 as the projections
    wrote them, slices of one buffer's rows among them.  inv_freq: fp64
    [rot_dim / 2] on the device, None for no rotation.  Tokens whose slot is
    outside the cache (-1) are left out, their rows of q_out as well."""
    n, Hkv, P, D = _caches(k_cache, v_cache)
    dev = _device(k_cache, "k_cache")
    if q.dim() != 3:
        raise ValueError("q must be [T, Hq, D]")
    T, Hq = q.shape[0], q.shape[1]
    src = _DTYPES.get(q.dtype)
    if src is None or k.dtype is not q.dtype or v.dtype is not q.dtype:
        raise TypeError("q, k and v must be float32, float16 or bfloat16, all the same")
    rot, freq = 0, None
    if inv_freq is not None:
        if inv_freq.dtype is not torch.float64 or not inv_freq.is_contiguous():
            raise TypeError("inv_freq must be contiguous float64")
        rot, freq = 2 * inv_freq.numel(), _on(inv_freq, "inv_freq", dev).data_ptr()
    if q_out is None:
        q_out = _new((T, Hq, D), k_cache.dtype, k_cache, stream)
    elif q_out.dtype is not k_cache.dtype:
        raise TypeError("q_out must have the caches' type")
    for t, name in ((q, "q"), (k, "k"), (v, "v"), (v_cache, "v_cache"), (q_out, "q_out")):
        _on(t, name, dev)
    qp, qs = _rows(q, "q", T, Hq, D)
    kp, ks = _rows(k, "k", T, Hkv, D)
    vp, vs = _rows(v, "v", T, Hkv, D)
    op, os = _rows(q_out, "q_out", T, Hq, D)
    _launch(_lib.load().ifx_rope_append, "ifx_rope_append", dev, stream, qp, qs, kp, ks, vp, vs, src,
            _i32(positions, "positions", T, dev), _i32(slots, "slots", T, dev), freq, rot,
            1 if interleaved else 0, T, Hq, Hkv, D, op, os, k_cache.data_ptr(), v_cache.data_ptr(),
            _DTYPES[k_cache.dtype], n, P)
    return q_out


def _out(q, out, out_dtype, stream):
    want = out_dtype or (q.dtype if out is None else out.dtype)
    if want not in _DTYPES or (out is not None and out.dtype is not want):
        raise TypeError("out must be float32, float16 or bfloat16, and of out_dtype if that is given")
    return _new(q.shape, want, q, stream) if out is None else out


def paged_workspace_bytes(B, T, Hq, Hkv, head_dim, max_q, max_kv):
    """Bytes of workspace that paged_attention needs for this shape (0: none;
    WORKSPACE_BYTES is enough for all)."""
    return int(_lib.load().ifx_attn_paged_workspace_bytes(
        _count(B, "B"), _count(T, "T"), _count(Hq, "Hq"), _count(Hkv, "Hkv"),
        _count(head_dim, "head_dim"), _count(max_q, "max_q"), _count(max_kv, "max_kv")))


def paged_attention(q, k_cache, v_cache, block_table, cu_q, kv_len, max_q, max_kv, scale=None,
                    window=0, out=None, out_dtype=None, workspace=None, stream=None):
    """Attention of the new tokens q [T, Hq, D] over the paged cache, which
    holds them already (ifx_attn_paged).  cu_q [B + 1]: the requests' first
    rows; kv_len [B]: their tokens, the new ones included; max_q, max_kv: bounds
    of a request's rows (those past max_q may be left out) and tokens.  A query
    sees its own position and what is before it, the last `window` keys of it
    where window > 0.  scale: head_dim ** -0.5 if None.
    Returns out [T, Hq, D] (out_dtype: fp32, fp16 or bf16, q's type if None);
    its rows from cu_q[B] on are left as they were.  workspace: see
    `workspace` and paged_workspace_bytes."""
    n, Hkv, P, D = _caches(k_cache, v_cache)
    dev = _device(q, "q")
    if q.dim() != 3:
        raise ValueError("q must be [T, Hq, D]")
    if q.dtype is not k_cache.dtype:
        raise TypeError("q must have the caches' type")
    T, Hq = q.shape[0], q.shape[1]
    B = kv_len.numel()
    if block_table.dim() != 2 or block_table.shape[0] != B:
        raise ValueError("block_table must be [B, pages]")
    W = block_table.shape[1]
    out = _out(q, out, out_dtype, stream)
    for t, name in ((k_cache, "k_cache"), (v_cache, "v_cache"), (out, "out")):
        _on(t, name, dev)
    qp, qs = _rows(q, "q", T, Hq, D)
    op, os = _rows(out, "out", T, Hq, D)
    wp, wn = None, 0
    if workspace is not None:
        if not workspace.is_contiguous():
            raise ValueError("workspace must be contiguous")
        wp, wn = _on(workspace, "workspace", dev).data_ptr(), workspace.nbytes
    _launch(_lib.load().ifx_attn_paged, "ifx_attn_paged", dev, stream, qp, qs, _DTYPES[q.dtype],
            k_cache.data_ptr(), v_cache.data_ptr(), n, P,
            _i32(block_table, "block_table", B * W, dev), W, _i32(cu_q, "cu_q", B + 1, dev),
            _i32(kv_len, "kv_len", B, dev), B, T, Hq, Hkv, D, _count(max_q, "max_q"),
            _count(max_kv, "max_kv"), D ** -0.5 if scale is None else scale,
            _count(window, "window"), op, os, _DTYPES[out.dtype], wp, wn)
    return out


def prompt_attention(q, k, v, cu_len, max_len, causal=True, window=0, scale=None, out=None,
                     out_dtype=None, stream=None):
    """Attention over whole prompts packed one after the other, without a cache
    (ifx_attn_prompt): q [T, Hq, D], k and v [T, Hkv, D] (fp16 or bf16), rows
    cu_len[b] .. cu_len[b + 1] - 1 are prompt b, max_len bounds the lengths
    (checked to be positive, no launch depends on it).
    A row sees its prompt's rows; where causal those up to its own, the last
    `window` of them where window > 0.  Returns out [T, Hq, D] (out_dtype:
    fp32, fp16 or bf16, q's type if None)."""
    dev = _device(q, "q")
    if q.dim() != 3 or k.dim() != 3:
        raise ValueError("q, k and v must be [T, heads, D]")
    if q.dtype not in _ELEMS or k.dtype is not q.dtype or v.dtype is not q.dtype:
        raise TypeError("q, k and v must be float16 or bfloat16, all the same")
    T, Hq, D = q.shape
    Hkv, B = k.shape[1], cu_len.numel() - 1
    out = _out(q, out, out_dtype, stream)
    for t, name in ((k, "k"), (v, "v"), (out, "out")):
        _on(t, name, dev)
    qp, qs = _rows(q, "q", T, Hq, D)
    kp, ks = _rows(k, "k", T, Hkv, D)
    vp, vs = _rows(v, "v", T, Hkv, D)
    op, os = _rows(out, "out", T, Hq, D)
    _launch(_lib.load().ifx_attn_prompt, "ifx_attn_prompt", dev, stream, qp, qs, kp, ks, vp, vs,
            _DTYPES[q.dtype], _i32(cu_len, "cu_len", B + 1, dev), B, T, Hq, Hkv, D,
            _count(max_len, "max_len"), 1 if causal else 0, _count(window, "window"),
            D ** -0.5 if scale is None else scale, op, os, _DTYPES[out.dtype])
    return out
