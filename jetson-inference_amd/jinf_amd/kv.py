"""Drafted tokens and bounded KV caches (include/jinf/kv/kv_hip.h): attention of
a tree of drafted tokens over the cache, the accepted tokens' rows into the
caches, decode attention that adds up each position's attention weight, and the
eviction of the positions of least accumulated weight.

Caches are those of attention_decode, [n_seq, max_ctx, n_heads_kv * head_dim]
fp32 or fp16; accumulated weights are fp32 [n_seq, n_heads_kv, max_ctx].  Tensors
must live on the current HIP device; calls are enqueued on torch's current
stream and nothing synchronizes.  Each function raises JinfError for arguments
it cannot serve.
"""
import numpy as np
import torch

from ._lib import F16, F32, JINF_HIP_OK, lib
from .ops import JinfError

MAX_NODES = 256

# These calls take microseconds on the device, so what is checked on the way is
# checked with few Python operations.
_raw_stream = torch._C._cuda_getCurrentRawStream
_TYPES = {torch.float32: F32, torch.float16: F16}


def _device(names, *tensors):
    """The current device, which holds every given tensor (names: theirs, for the error)."""
    here = torch.cuda.current_device() if torch.cuda.is_initialized() else -2
    for i, t in enumerate(tensors):
        if t is not None and t.get_device() != here:
            name = names.split()[i]
            if not t.is_cuda:
                raise JinfError(f"{name} is not on the HIP device")
            raise JinfError(f"{name} is on {t.device}, the current device is "
                            f"cuda:{torch.cuda.current_device()}")
    return here


def _ints(name, t, *shape):
    """A contiguous int32 tensor of this shape."""
    if t.dtype is not torch.int32 or t.shape != shape or not t.is_contiguous():
        raise JinfError(f"{name} must be contiguous int32 {list(shape)}")


def _floats(name, t, *shape):
    """Strides of an fp32 tensor of this shape."""
    strides = t.stride()
    if t.dtype is not torch.float32 or t.shape != shape or (strides[-1] != 1 and t.numel()):
        raise JinfError(f"{name} must be fp32 {list(shape)}, contiguous in its last dimension")
    return strides


def _caches(k, v, names="k and v caches"):
    """Shape, strides and type code of a pair of caches or of rows for them."""
    shape, strides, code = k.shape, k.stride(), _TYPES.get(k.dtype)
    if (len(shape) != 3 or code is None or v.shape != shape or v.dtype is not k.dtype or
            v.stride() != strides or (strides[2] != 1 and k.numel())):
        raise JinfError(f"{names} must be two fp32 or fp16 [n_seq, positions, n_heads_kv * head_dim] "
                        "tensors of one type and layout")
    return shape, strides, code


def _head_dim(width, n_heads_kv):
    if n_heads_kv <= 0 or width % n_heads_kv or width == 0:
        raise JinfError("cache width must be n_heads_kv * head_dim")
    return width // n_heads_kv


def _space(workspace, nbytes, device):
    """The caller's workspace, or one of this call's own."""
    if workspace is None:
        return torch.empty(max(nbytes(), 16), dtype=torch.uint8, device=device)
    if workspace.dtype is not torch.uint8 or not workspace.is_contiguous():
        raise JinfError("workspace must be a contiguous uint8 tensor")
    return workspace


def _ptr(t):
    return None if t is None else t.data_ptr()


def _check(rc, name):
    if rc != JINF_HIP_OK:
        raise JinfError(f"{name} returned status {rc}")


def tree_mask(parents, device="cuda"):
    """Mask words of trees given by parents: parents [n_seq, nodes] integers on the
    host, parents[s][i] < i the node that node i follows, or -1 for one that
    follows the cached context.  Node i attends to itself and its ancestors.
    Returns int64 [n_seq, nodes, ceil(nodes / 64)]."""
    p = np.asarray(parents, dtype=np.int64)
    if p.ndim != 2 or not 0 < p.shape[1] <= MAX_NODES:
        raise JinfError(f"parents must be [n_seq, nodes], 1 to {MAX_NODES} nodes")
    n, T = p.shape
    if np.any(p < -1) or np.any(p >= np.arange(T)):
        raise JinfError("a node's parent must come before it (or be -1)")
    words = (T + 63) // 64
    bits = np.zeros((n, T + 1, words * 64), dtype=np.uint8)  # row T: the context's own, no node
    rows = np.arange(n)
    for i in range(T):
        bits[:, i] = bits[rows, p[:, i]]
        bits[:, i, i] = 1
    packed = np.packbits(bits[:, :T], axis=-1, bitorder="little")
    return torch.from_numpy(packed.view(np.int64).copy()).to(device)


def attention_tree_workspace(n_seq, max_nodes, n_heads, n_heads_kv, head_dim, max_ctx,
                             device="cuda"):
    """A workspace for attention_tree calls of up to these sizes."""
    nbytes = lib().jinf_attention_tree_workspace_bytes(n_seq, max_nodes, n_heads, n_heads_kv,
                                                       head_dim, max_ctx)
    return torch.empty(max(nbytes, 16), dtype=torch.uint8, device=device)


def attention_tree(q, k_cache, v_cache, lens, k_draft, v_draft, mask, n_heads, n_heads_kv,
                   n_nodes=None, scale=0.0, out=None, workspace=None):
    """Attention of drafted tokens: node (s, i) over the cached positions t < lens[s]
    and the nodes whose bits its mask row holds (tree_mask).  q fp32 [n_seq,
    nodes, n_heads * hd]; k_draft, v_draft [n_seq, nodes, n_heads_kv * hd] fp32 or
    fp16, used as the cache would hold them; mask int64 [n_seq, nodes,
    ceil(nodes / 64)]; n_nodes int32 [n_seq]: nodes of each sequence (None: all).
    Rows past them stay as they were in `out` (zeros in a new one).  Returns out
    fp32 like q."""
    (n_seq, max_ctx, width), kst, kt = _caches(k_cache, v_cache)
    dshape, dst, dt = _caches(k_draft, v_draft, "k and v drafts")
    hd, nodes = _head_dim(width, n_heads_kv), dshape[1]
    here = _device("q k_cache v_cache lens k_draft v_draft mask n_nodes out workspace", q, k_cache,
                   v_cache, lens, k_draft, v_draft, mask, n_nodes, out, workspace)
    if dshape != (n_seq, nodes, width):
        raise JinfError("drafts must be [n_seq, nodes, n_heads_kv * head_dim]")
    qst = _floats("q", q, n_seq, nodes, n_heads * hd)
    if (mask.dtype is not torch.int64 or mask.shape != (n_seq, nodes, (nodes + 63) // 64) or
            not mask.is_contiguous()):
        raise JinfError("mask must be contiguous int64 [n_seq, nodes, ceil(nodes / 64)]")
    _ints("lens", lens, n_seq)
    if n_nodes is not None:
        _ints("n_nodes", n_nodes, n_seq)
    if out is None:
        make = torch.empty if n_nodes is None else torch.zeros
        out = make((n_seq, nodes, n_heads * hd), dtype=torch.float32, device=q.device)
    ost = _floats("out", out, n_seq, nodes, n_heads * hd)
    L = lib()
    workspace = _space(workspace, lambda: L.jinf_attention_tree_workspace_bytes(
        n_seq, nodes, n_heads, n_heads_kv, hd, max_ctx), q.device)
    _check(L.jinf_attention_tree(
        out.data_ptr(), ost[1], ost[0], q.data_ptr(), qst[1], qst[0], k_cache.data_ptr(),
        v_cache.data_ptr(), kt, kst[1], kst[0], lens.data_ptr(), k_draft.data_ptr(),
        v_draft.data_ptr(), dt, dst[1], dst[0], mask.data_ptr(), _ptr(n_nodes), nodes, n_seq,
        max_ctx, hd, n_heads, n_heads_kv, scale, workspace.data_ptr(), workspace.numel(),
        _raw_stream(here)), "jinf_attention_tree")
    return out


def cache_append(k_cache, v_cache, lens, k_rows, v_rows, n_heads_kv, index=None, counts=None,
                 weights=None, lens_out=None):
    """Appends row index[s, a] (row a: None) of k_rows / v_rows [n_seq, rows,
    n_heads_kv * hd] (fp32 or fp16) to sequence s's caches at lens[s] + a, for a <
    counts[s] (every one: None); rows past the cache's end are dropped, an index
    outside the rows stores zeros.  weights: the new positions' accumulated
    weights are set to 0.  Returns the new lengths (lens_out; not lens itself)."""
    (n_seq, max_ctx, width), kst, kt = _caches(k_cache, v_cache)
    (rn, rows, rwidth), rst, rt = _caches(k_rows, v_rows, "k and v rows")
    hd = _head_dim(width, n_heads_kv)
    lens_out = torch.empty_like(lens) if lens_out is None else lens_out
    here = _device("k_cache v_cache lens k_rows v_rows index counts weights lens_out", k_cache,
                   v_cache, lens, k_rows, v_rows, index, counts, weights, lens_out)
    if rn != n_seq or rwidth != width:
        raise JinfError("rows must be [n_seq, rows, n_heads_kv * head_dim]")
    _ints("lens", lens, n_seq)
    _ints("lens_out", lens_out, n_seq)
    take = rows
    if index is not None:
        take = index.shape[1] if index.dim() == 2 else -1
        _ints("index", index, n_seq, take)
    if counts is not None:
        _ints("counts", counts, n_seq)
    wst = (0, 0) if weights is None else _floats("weights", weights, n_seq, n_heads_kv, max_ctx)
    _check(lib().jinf_cache_append(
        k_cache.data_ptr(), v_cache.data_ptr(), kt, kst[1], kst[0], _ptr(weights), wst[1], wst[0],
        lens.data_ptr(), lens_out.data_ptr(), k_rows.data_ptr(), v_rows.data_ptr(), rt, rst[1],
        rst[0], rows, _ptr(index), _ptr(counts), take, n_seq, max_ctx, hd, n_heads_kv,
        _raw_stream(here)), "jinf_cache_append")
    return lens_out


def attention_scored_workspace(n_seq, n_heads, n_heads_kv, head_dim, max_ctx, device="cuda"):
    """A workspace for attention_decode_scored calls of up to these sizes."""
    nbytes = lib().jinf_attention_scored_workspace_bytes(n_seq, n_heads, n_heads_kv, head_dim,
                                                         max_ctx)
    return torch.empty(max(nbytes, 16), dtype=torch.uint8, device=device)


def attention_decode_scored(q, k_cache, v_cache, lens, weights, n_heads, n_heads_kv, scale=0.0,
                            out=None, workspace=None):
    """attention_decode that also adds each position's attention weight, summed over
    the query heads of a kv head, to weights fp32 [n_seq, n_heads_kv, max_ctx] in
    place.  Returns out fp32 [n_seq, n_heads * hd]."""
    (n_seq, max_ctx, width), kst, kt = _caches(k_cache, v_cache)
    hd = _head_dim(width, n_heads_kv)
    here = _device("q k_cache v_cache lens weights out workspace", q, k_cache, v_cache, lens,
                   weights, out, workspace)
    qst = _floats("q", q, n_seq, n_heads * hd)
    wst = _floats("weights", weights, n_seq, n_heads_kv, max_ctx)
    _ints("lens", lens, n_seq)
    if out is None:
        out = torch.empty((n_seq, n_heads * hd), dtype=torch.float32, device=q.device)
    ost = _floats("out", out, n_seq, n_heads * hd)
    L = lib()
    workspace = _space(workspace, lambda: L.jinf_attention_scored_workspace_bytes(
        n_seq, n_heads, n_heads_kv, hd, max_ctx), q.device)
    _check(L.jinf_attention_decode_scored(
        out.data_ptr(), ost[0], q.data_ptr(), qst[0], k_cache.data_ptr(), v_cache.data_ptr(), kt,
        kst[1], kst[0], weights.data_ptr(), wst[1], wst[0], lens.data_ptr(), n_seq, max_ctx, hd,
        n_heads, n_heads_kv, scale, workspace.data_ptr(), workspace.numel(), _raw_stream(here)),
        "jinf_attention_decode_scored")
    return out


def cache_evict_workspace(n_seq, n_heads_kv, budget, device="cuda"):
    """A workspace for cache_evict calls of up to these sizes."""
    nbytes = lib().jinf_cache_evict_workspace_bytes(n_seq, n_heads_kv, budget)
    return torch.empty(max(nbytes, 16), dtype=torch.uint8, device=device)


def cache_evict(k_cache, v_cache, weights, lens, n_heads_kv, budget, n_first=0, n_recent=0,
                k_out=None, v_out=None, weights_out=None, lens_out=None, kept=None,
                workspace=None):
    """Takes each (sequence, kv head) down to `budget` positions: the first n_first, the
    last n_recent and, of the others, those of largest accumulated weight (the
    lowest position among equals).  Kept rows move together in their order, in
    place, or to k_out / v_out / weights_out (all three given, of the inputs' layout
    with min(budget, max_ctx) positions or more).  kept: int32 [n_seq, n_heads_kv,
    budget] receives the old positions (-1 past the new length).  Returns the new
    lengths min(lens, budget) (lens_out; may be lens)."""
    (n_seq, max_ctx, width), kst, kt = _caches(k_cache, v_cache)
    hd = _head_dim(width, n_heads_kv)
    wst = _floats("weights", weights, n_seq, n_heads_kv, max_ctx)
    if k_out is None and v_out is None and weights_out is None:
        k_out, v_out, weights_out, ost, wost = k_cache, v_cache, weights, kst, wst
    elif k_out is None or v_out is None or weights_out is None:
        raise JinfError("k_out, v_out and weights_out go together")
    else:
        (on, rows, owidth), ost, ot = _caches(k_out, v_out, "k and v outputs")
        if on != n_seq or owidth != width or ot != kt:
            raise JinfError("outputs must have the caches' type, sequences and width")
        if rows < min(budget, max_ctx):
            raise JinfError("outputs hold fewer positions than stay")
        wost = _floats("weights_out", weights_out, n_seq, n_heads_kv, rows)
    lens_out = torch.empty_like(lens) if lens_out is None else lens_out
    here = _device("k_cache v_cache weights lens k_out v_out weights_out lens_out kept workspace",
                   k_cache, v_cache, weights, lens, k_out, v_out, weights_out, lens_out, kept,
                   workspace)
    _ints("lens", lens, n_seq)
    _ints("lens_out", lens_out, n_seq)
    if kept is not None:
        _ints("kept", kept, n_seq, n_heads_kv, budget)
    L = lib()
    workspace = _space(workspace, lambda: L.jinf_cache_evict_workspace_bytes(
        n_seq, n_heads_kv, budget), k_cache.device)
    _check(L.jinf_cache_evict(
        k_out.data_ptr(), v_out.data_ptr(), ost[1], ost[0], k_cache.data_ptr(), v_cache.data_ptr(),
        kt, kst[1], kst[0], weights_out.data_ptr(), wost[1], wost[0], weights.data_ptr(), wst[1],
        wst[0], lens.data_ptr(), lens_out.data_ptr(), _ptr(kept), budget, n_first, n_recent, n_seq,
        max_ctx, hd, n_heads_kv, workspace.data_ptr(), workspace.numel(), _raw_stream(here)),
        "jinf_cache_evict")
    return lens_out
