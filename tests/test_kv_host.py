"""The drafted-token and bounded-cache entry points without a GPU: the header's
declarations are exported and bound, bad arguments are refused on the host
before any launch, and tree_mask."""
import ctypes
import os
import re

import numpy as np
import pytest
import torch

import jinf_amd
import kv_ref
from jinf_amd import _lib

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HEADER = os.path.join(ROOT, "include", "jinf", "kv", "kv_hip.h")
OK, INVALID = _lib.JINF_HIP_OK, _lib.JINF_HIP_ERR_INVALID
FAKE = 0x100000  # never dereferenced: every call below ends on the host


def test_header_is_exported_and_bound():
    src = re.sub(r"/\*.*?\*/", "", open(HEADER).read(), flags=re.S)
    assert not re.search(r"#include\s*[<\"](hip|cuda)", src)
    decl = {m.group(1): m.group(2).count(",") + 1
            for m in re.finditer(r"\b(jinf_\w+)\s*\(([^)]*)\)\s*;", src)}
    assert len(decl) == 7
    for name, n in decl.items():
        assert hasattr(jinf_amd.lib(), name), name
        assert len(_lib.SIGNATURES[name][1]) == n, name


TREE = dict(out=FAKE, ld_out=512, ld_out_seq=4 * 512, q=FAKE, ld_q=512, ld_q_seq=4 * 512,
            k_cache=FAKE, v_cache=FAKE, kv_type=1, ld_pos=128, ld_seq=128 * 32, lens=FAKE,
            k_draft=FAKE, v_draft=FAKE, draft_type=0, ld_draft=128, ld_draft_seq=4 * 128, mask=FAKE,
            n_nodes=None, max_nodes=4, n_seq=2, max_ctx=32, head_dim=64, n_heads=8, n_heads_kv=2,
            scale=0.0, workspace=None, workspace_bytes=0, stream=None)
APPEND = dict(k_cache=FAKE, v_cache=FAKE, kv_type=1, ld_pos=128, ld_seq=128 * 32, weights=FAKE,
              ld_w=32, ld_w_seq=64, lens=FAKE, lens_out=FAKE + 64, k_rows=FAKE, v_rows=FAKE,
              rows_type=0, ld_rows=128, ld_rows_seq=512, n_rows=4, index=None, counts=None, n_take=4,
              n_seq=2, max_ctx=32, head_dim=64, n_heads_kv=2, stream=None)
SCORED = dict(out=FAKE, ld_out=512, q=FAKE, ld_q=512, k_cache=FAKE, v_cache=FAKE, kv_type=1,
              ld_pos=128, ld_seq=128 * 32, weights=FAKE, ld_w=32, ld_w_seq=64, lens=FAKE, n_seq=2,
              max_ctx=32, head_dim=64, n_heads=8, n_heads_kv=2, scale=0.0, workspace=FAKE,
              workspace_bytes=1 << 30, stream=None)
EVICT = dict(k_out=FAKE, v_out=FAKE + (1 << 20), ld_pos_out=128, ld_seq_out=128 * 32, k_cache=FAKE,
             v_cache=FAKE + (1 << 20), kv_type=1, ld_pos=128, ld_seq=128 * 32, weights_out=FAKE,
             ld_wo=32, ld_wo_seq=64, weights=FAKE, ld_w=32, ld_w_seq=64, lens=FAKE, lens_out=FAKE,
             kept=None, budget=16, n_first=2, n_recent=4, n_seq=2, max_ctx=32, head_dim=64,
             n_heads_kv=2, workspace=FAKE, workspace_bytes=1 << 30, stream=None)
FN = {"tree": ("jinf_attention_tree", TREE), "append": ("jinf_cache_append", APPEND),
      "scored": ("jinf_attention_decode_scored", SCORED), "evict": ("jinf_cache_evict", EVICT)}


def call(fn, **changes):
    name, args = FN[fn]
    assert set(changes) <= set(args)
    return getattr(jinf_amd.lib(), name)(*{**args, **changes}.values())


@pytest.mark.parametrize("fn,changes", [
    *[(f, {"n_seq": -1}) for f in FN],
    *[(f, {"n_seq": 70000}) for f in FN],
    *[(f, {"max_ctx": -1}) for f in FN],
    *[(f, {"max_ctx": (1 << 30) + 1, "ld_seq": 1 << 40}) for f in FN],
    *[(f, {"head_dim": 0}) for f in FN],
    *[(f, {"head_dim": 1025}) for f in FN],
    *[(f, {"n_heads_kv": 0}) for f in FN],
    *[(f, {"kv_type": 2}) for f in FN],
    *[(f, {"lens": None}) for f in FN],
    *[(f, {"lens": FAKE + 2}) for f in FN],
    *[(f, {"k_cache": None}) for f in FN],
    *[(f, {"v_cache": FAKE + 1}) for f in FN],
    *[(f, {"ld_pos": 127}) for f in FN],
    *[(f, {"ld_seq": 128 * 31}) for f in FN],
    ("append", {"ld_seq": 0}), ("evict", {"ld_seq": 0, "ld_seq_out": 0}),
    *[(f, {"n_heads": 7}) for f in ("tree", "scored")],
    *[(f, {"scale": s}) for f in ("tree", "scored") for s in (-1.0, float("nan"), float("inf"))],
    *[(f, {"q": None}) for f in ("tree", "scored")],
    *[(f, {"out": None}) for f in ("tree", "scored")],
    *[(f, {"q": FAKE + 2}) for f in ("tree", "scored")],
    *[(f, {"ld_q": 511}) for f in ("tree", "scored")],
    *[(f, {"ld_out": 511}) for f in ("tree", "scored")],
    ("tree", {"max_nodes": 257}), ("tree", {"max_nodes": -1}), ("tree", {"mask": None}),
    ("tree", {"mask": FAKE + 4}), ("tree", {"k_draft": None}), ("tree", {"v_draft": FAKE + 2}),
    ("tree", {"draft_type": 3}), ("tree", {"ld_draft": 127}), ("tree", {"ld_q_seq": 2047}),
    ("tree", {"ld_out_seq": 2047}), ("tree", {"ld_draft_seq": 511}), ("tree", {"n_nodes": FAKE + 1}),
    ("tree", {"workspace": FAKE + 8, "workspace_bytes": 64}),
    *[(f, {"ld_w": 31}) for f in ("append", "scored", "evict")],
    *[(f, {"ld_w_seq": 63}) for f in ("append", "scored", "evict")],
    *[(f, {"weights": FAKE + 2}) for f in ("append", "scored")],
    ("scored", {"weights": None}), ("scored", {"workspace": None}), ("scored", {"workspace_bytes": 8}),
    ("scored", {"workspace": FAKE + 4}),
    ("append", {"lens_out": FAKE}), ("append", {"n_take": 5}), ("append", {"n_take": -1}),
    ("append", {"n_rows": -1}), ("append", {"k_rows": None}), ("append", {"rows_type": 2}),
    ("append", {"ld_rows": 127}), ("append", {"v_rows": FAKE + 2}),
    ("evict", {"budget": -1}), ("evict", {"n_first": -1}), ("evict", {"n_recent": -1}),
    ("evict", {"n_first": 13}), ("evict", {"workspace": None}), ("evict", {"workspace_bytes": 8}),
    ("evict", {"k_out": None}), ("evict", {"weights": None}),
    # part in place, part not; in place with other strides
    ("evict", {"v_out": FAKE + (1 << 24)}), ("evict", {"weights_out": FAKE + (1 << 24)}),
    ("evict", {"ld_pos_out": 136}), ("evict", {"ld_seq_out": 128 * 40}), ("evict", {"ld_wo": 40}),
    # apart, but overlapping the input, or too short
    ("evict", {"k_out": FAKE + 256, "v_out": FAKE + (1 << 24), "weights_out": FAKE + (1 << 24)}),
    ("evict", {"k_out": FAKE + (1 << 23), "v_out": FAKE + (1 << 20) - 64,
               "weights_out": FAKE + (1 << 24)}),
    ("evict", {"k_out": FAKE + (1 << 23), "v_out": FAKE + (1 << 24), "weights_out": FAKE + 4}),
    ("evict", {"k_out": FAKE + (1 << 23), "v_out": FAKE + (1 << 24), "ld_seq_out": 128 * 15,
               "weights_out": FAKE + (1 << 25)}),
    ("evict", {"k_out": FAKE + (1 << 23), "v_out": FAKE + (1 << 24), "ld_wo": 15,
               "weights_out": FAKE + (1 << 25)}),
])
def test_refused_on_the_host(fn, changes):
    assert call(fn, **changes) == INVALID


@pytest.mark.parametrize("fn", list(FN))
def test_no_sequences_is_ok(fn):
    assert call(fn, n_seq=0) == OK


def test_no_nodes_is_ok():
    assert call("tree", max_nodes=0) == OK


def test_workspace_sizes_of_empty_shapes():
    L = jinf_amd.lib()
    assert L.jinf_attention_tree_workspace_bytes(0, 4, 8, 2, 64, 32) == 0
    assert L.jinf_attention_scored_workspace_bytes(2, 0, 2, 64, 32) == 0
    assert L.jinf_cache_evict_workspace_bytes(2, 2, 0) == 0


def test_host_tensors_are_refused():
    k = torch.zeros(1, 8, 128)
    lens = torch.ones(1, dtype=torch.int32)
    q, w = torch.zeros(1, 512), torch.zeros(1, 2, 8)
    mask = torch.ones(1, 1, 1, dtype=torch.int64)
    for fn in (lambda: jinf_amd.attention_tree(q[None], k, k, lens, k[:, :1], k[:, :1], mask, 8, 2),
               lambda: jinf_amd.attention_decode_scored(q, k, k, lens, w, 8, 2),
               lambda: jinf_amd.cache_append(k, k, lens, k[:, :1], k[:, :1], 2),
               lambda: jinf_amd.cache_evict(k, k, w, lens, 2, 4)):
        with pytest.raises(jinf_amd.JinfError, match="HIP device"):
            fn()


def test_mismatched_caches_are_refused():
    k, lens = torch.zeros(1, 8, 128), torch.ones(1, dtype=torch.int32)
    w = torch.zeros(1, 2, 8)
    for a, b in ((k, k.half()), (k, k[:, :4]), (k[0], k[0]), (k, k.transpose(1, 2))):
        with pytest.raises(jinf_amd.JinfError):
            jinf_amd.cache_evict(a, b, w, lens, 2, 4)
    with pytest.raises(jinf_amd.JinfError):
        jinf_amd.cache_evict(k, k, w, lens, 3, 4)
    with pytest.raises(jinf_amd.JinfError):
        jinf_amd.cache_evict(k, k, w, lens, 2, 4, k_out=k.clone())


@pytest.mark.parametrize("T", [1, 7, 64, 65, 256])
def test_tree_mask(T):
    r = np.random.default_rng(T)
    parents = np.stack([[r.integers(-1, i) if i else -1 for i in range(T)] for _ in range(3)])
    got = kv_ref.mask_bits(jinf_amd.tree_mask(parents, device="cpu"))
    for s in range(3):
        for i in range(T):
            want, at = {i}, parents[s, i]
            while at >= 0:
                want.add(int(at))
                at = parents[s, at]
            assert set(np.flatnonzero(got[s, i])) == want


@pytest.mark.parametrize("parents", [[[0]], [[-1, 1]], [[-2]], [[-1, 5]], [-1, 0], [[]],
                                     np.full((1, 257), -1)])
def test_tree_mask_refusals(parents):
    with pytest.raises(jinf_amd.JinfError):
        jinf_amd.tree_mask(parents, device="cpu")


def test_reference_keep_orders_ties_and_nan():
    w = np.array([0.0, 3.0, -0.0, np.nan, 3.0, np.inf, 0.0, 3.0])
    assert list(kv_ref.keep(w, 8, 3, 0, 0)) == [1, 3, 5]
    assert list(kv_ref.keep(w, 8, 5, 1, 1)) == [0, 1, 3, 5, 7]
    assert list(kv_ref.keep(w, 3, 3, 1, 1)) == [0, 1, 2]
    assert ctypes.sizeof(ctypes.c_void_p) == 8
