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

from ._lib import lib
from .ops import JinfError, _act, _check, _ptr, _stream

MAX_NODES = 256


def _here(**tensors):
    """Every given tensor on the current device."""
    for name, t in tensors.items():
        if t is None:
            continue
        if not t.is_cuda:
            raise JinfError(f"{name} is not on the HIP device")
        if t.device.index != torch.cuda.current_device():
            raise JinfError(f"{name} is on {t.device}, the current device is "
                            f"cuda:{torch.cuda.current_device()}")


def _ints(name, t, *shape):
    """A contiguous int32 tensor of this shape (None passes)."""
    if t is None:
        return
    if t.dtype != torch.int32 or tuple(t.shape) != shape or not t.is_contiguous():
        raise JinfError(f"{name} must be contiguous int32 {list(shape)}")


def _floats(name, t, *shape):
    if t.dtype != torch.float32 or tuple(t.shape) != shape or (t.numel() and t.stride(-1) != 1):
        raise JinfError(f"{name} must be fp32 {list(shape)}, contiguous in its last dimension")


def _caches(k, v, n_heads_kv, names="k and v caches"):
    """(n_seq, max_ctx, head_dim) of a pair of caches."""
    if (k.dim() != 3 or k.shape != v.shape or k.dtype != v.dtype or k.stride() != v.stride() or
            (k.numel() and k.stride(2) != 1)):
        raise JinfError(f"{names} must be two [n_seq, positions, n_heads_kv * head_dim] tensors of "
                        "one type and layout")
    if n_heads_kv <= 0 or k.shape[2] % n_heads_kv or k.shape[2] == 0:
        raise JinfError("cache width must be n_heads_kv * head_dim")
    return k.shape[0], k.shape[1], k.shape[2] // n_heads_kv


def _space(workspace, nbytes, device):
    """The caller's workspace, or one of this call's own."""
    if workspace is None:
        workspace = torch.empty(max(nbytes, 16), dtype=torch.uint8, device=device)
    elif workspace.dtype != torch.uint8 or not workspace.is_contiguous():
        raise JinfError("workspace must be a contiguous uint8 tensor")
    return workspace


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
    n_seq, max_ctx, hd = _caches(k_cache, v_cache, n_heads_kv)
    nodes = q.shape[1] if q.dim() == 3 else -1
    _here(q=q, k_cache=k_cache, v_cache=v_cache, lens=lens, k_draft=k_draft, v_draft=v_draft,
          mask=mask, n_nodes=n_nodes, out=out, workspace=workspace)
    _floats("q", q, n_seq, nodes, n_heads * hd)
    dn, dt, _ = _caches(k_draft, v_draft, n_heads_kv, "k and v drafts")
    if (dn, dt, k_draft.shape[2]) != (n_seq, nodes, k_cache.shape[2]):
        raise JinfError("drafts must be [n_seq, nodes, n_heads_kv * head_dim]")
    if (mask.dtype != torch.int64 or tuple(mask.shape) != (n_seq, nodes, (nodes + 63) // 64) or
            not mask.is_contiguous()):
        raise JinfError("mask must be contiguous int64 [n_seq, nodes, ceil(nodes / 64)]")
    _ints("lens", lens, n_seq)
    _ints("n_nodes", n_nodes, n_seq)
    if out is None:
        make = torch.empty if n_nodes is None else torch.zeros
        out = make((n_seq, nodes, n_heads * hd), dtype=torch.float32, device=q.device)
    _floats("out", out, n_seq, nodes, n_heads * hd)
    workspace = _space(workspace, lib().jinf_attention_tree_workspace_bytes(
        n_seq, nodes, n_heads, n_heads_kv, hd, max_ctx), q.device)
    _check(lib().jinf_attention_tree(
        _ptr(out), out.stride(1), out.stride(0), _ptr(q), q.stride(1), q.stride(0), _ptr(k_cache),
        _ptr(v_cache), _act(k_cache), k_cache.stride(1), k_cache.stride(0), _ptr(lens),
        _ptr(k_draft), _ptr(v_draft), _act(k_draft), k_draft.stride(1), k_draft.stride(0),
        _ptr(mask), _ptr(n_nodes), nodes, n_seq, max_ctx, hd, n_heads, n_heads_kv, float(scale),
        _ptr(workspace), workspace.numel(), _stream()), "jinf_attention_tree")
    return out


def cache_append(k_cache, v_cache, lens, k_rows, v_rows, n_heads_kv, index=None, counts=None,
                 weights=None, lens_out=None):
    """Appends row index[s, a] (row a: None) of k_rows / v_rows [n_seq, rows,
    n_heads_kv * hd] (fp32 or fp16) to sequence s's caches at lens[s] + a, for a <
    counts[s] (every one: None); rows past the cache's end are dropped, an index
    outside the rows stores zeros.  weights: the new positions' accumulated
    weights are set to 0.  Returns the new lengths (lens_out; not lens itself)."""
    n_seq, max_ctx, hd = _caches(k_cache, v_cache, n_heads_kv)
    rn, rows, _ = _caches(k_rows, v_rows, n_heads_kv, "k and v rows")
    if rn != n_seq or k_rows.shape[2] != k_cache.shape[2]:
        raise JinfError("rows must be [n_seq, rows, n_heads_kv * head_dim]")
    take = rows if index is None else index.shape[-1]
    lens_out = torch.empty_like(lens) if lens_out is None else lens_out
    _here(k_cache=k_cache, v_cache=v_cache, lens=lens, k_rows=k_rows, v_rows=v_rows, index=index,
          counts=counts, weights=weights, lens_out=lens_out)
    _ints("lens", lens, n_seq)
    _ints("lens_out", lens_out, n_seq)
    _ints("index", index, n_seq, take)
    _ints("counts", counts, n_seq)
    if weights is not None:
        _floats("weights", weights, n_seq, n_heads_kv, max_ctx)
    _check(lib().jinf_cache_append(
        _ptr(k_cache), _ptr(v_cache), _act(k_cache), k_cache.stride(1), k_cache.stride(0),
        _ptr(weights), weights.stride(1) if weights is not None else 0,
        weights.stride(0) if weights is not None else 0, _ptr(lens), _ptr(lens_out), _ptr(k_rows),
        _ptr(v_rows), _act(k_rows), k_rows.stride(1), k_rows.stride(0), rows, _ptr(index),
        _ptr(counts), take, n_seq, max_ctx, hd, n_heads_kv, _stream()), "jinf_cache_append")
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
    n_seq, max_ctx, hd = _caches(k_cache, v_cache, n_heads_kv)
    _here(q=q, k_cache=k_cache, v_cache=v_cache, lens=lens, weights=weights, out=out,
          workspace=workspace)
    _floats("q", q, n_seq, n_heads * hd)
    _floats("weights", weights, n_seq, n_heads_kv, max_ctx)
    _ints("lens", lens, n_seq)
    if out is None:
        out = torch.empty((n_seq, n_heads * hd), dtype=torch.float32, device=q.device)
    _floats("out", out, n_seq, n_heads * hd)
    workspace = _space(workspace, lib().jinf_attention_scored_workspace_bytes(
        n_seq, n_heads, n_heads_kv, hd, max_ctx), q.device)
    _check(lib().jinf_attention_decode_scored(
        _ptr(out), out.stride(0), _ptr(q), q.stride(0), _ptr(k_cache), _ptr(v_cache),
        _act(k_cache), k_cache.stride(1), k_cache.stride(0), _ptr(weights), weights.stride(1),
        weights.stride(0), _ptr(lens), n_seq, max_ctx, hd, n_heads, n_heads_kv, float(scale),
        _ptr(workspace), workspace.numel(), _stream()), "jinf_attention_decode_scored")
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
    n_seq, max_ctx, hd = _caches(k_cache, v_cache, n_heads_kv)
    given = [t is not None for t in (k_out, v_out, weights_out)]
    if any(given) != all(given):
        raise JinfError("k_out, v_out and weights_out go together")
    if not any(given):
        k_out, v_out, weights_out = k_cache, v_cache, weights
    on, rows, _ = _caches(k_out, v_out, n_heads_kv, "k and v outputs")
    if (on, k_out.shape[2], k_out.dtype) != (n_seq, k_cache.shape[2], k_cache.dtype):
        raise JinfError("outputs must have the caches' type, sequences and width")
    if rows < min(int(budget), max_ctx):
        raise JinfError("outputs hold fewer positions than stay")
    lens_out = torch.empty_like(lens) if lens_out is None else lens_out
    _here(k_cache=k_cache, v_cache=v_cache, weights=weights, lens=lens, k_out=k_out, v_out=v_out,
          weights_out=weights_out, lens_out=lens_out, kept=kept, workspace=workspace)
    _floats("weights", weights, n_seq, n_heads_kv, max_ctx)
    _floats("weights_out", weights_out, n_seq, n_heads_kv, rows)
    _ints("lens", lens, n_seq)
    _ints("lens_out", lens_out, n_seq)
    _ints("kept", kept, n_seq, n_heads_kv, int(budget))
    workspace = _space(workspace, lib().jinf_cache_evict_workspace_bytes(n_seq, n_heads_kv,
                                                                         int(budget)),
                       k_cache.device)
    _check(lib().jinf_cache_evict(
        _ptr(k_out), _ptr(v_out), k_out.stride(1), k_out.stride(0), _ptr(k_cache), _ptr(v_cache),
        _act(k_cache), k_cache.stride(1), k_cache.stride(0), _ptr(weights_out),
        weights_out.stride(1), weights_out.stride(0), _ptr(weights), weights.stride(1),
        weights.stride(0), _ptr(lens), _ptr(lens_out), _ptr(kept), int(budget), int(n_first),
        int(n_recent), n_seq, max_ctx, hd, n_heads_kv, _ptr(workspace), workspace.numel(),
        _stream()), "jinf_cache_evict")
    return lens_out
