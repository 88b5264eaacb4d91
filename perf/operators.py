"""The operators for drafted tokens and bounded KV caches, as measured cases of
plain values.

Kinds (a case's "kind"):
  tree    attention of a tree of drafted tokens over the cache and over each
          node's ancestors in the tree
  append  accepted tokens' K / V rows into the caches
  scored  one decode step's attention that also adds each cached position's
          attention weight to the position's running sum
  evict   the positions of smallest accumulated weight leave the caches

listed() holds fixed cases, draw(rng) makes further ones of the same ranges,
prepare/run are one user's program (own: through jinf_amd; otherwise the plain
form in torch), work() the bytes and operations a pass cannot do without,
exact() the same results in 64 bits.
"""
import math
import os
import sys

import numpy as np
import torch

own = False

# Attention widths: Llama-3-8B, Llama-3-70B and a small model with 64-wide heads.
M8B = {"n_heads": 32, "n_kv": 8, "head_dim": 128}
M70B = {"n_heads": 64, "n_kv": 8, "head_dim": 128}
M1B = {"n_heads": 32, "n_kv": 8, "head_dim": 64}


def listed():
    return [
        # One user's chat: a small tree of drafted tokens over a short context.
        dict(name="tree_1seq_8b", kind="tree", n_seq=1, nodes=7, ctx=333, kv="f16", draft="f32",
             **M8B),
        # A server's ragged batch, trees of up to 25 nodes.
        dict(name="tree_16seq_8b", kind="tree", n_seq=16, nodes=25, ctx=4096, kv="f16",
             draft="f32", **M8B),
        # Four long documents, the widest trees a batch decoder's step holds.
        dict(name="tree_4seq_70b_long", kind="tree", n_seq=4, nodes=64, ctx=32768, kv="f16",
             draft="f16", **M70B),
        # A small model over the fp32 cache the reference engine keeps.
        dict(name="tree_5seq_1b_f32", kind="tree", n_seq=5, nodes=13, ctx=1999, kv="f32",
             draft="f32", **M1B),
        # The accepted path (up to 5 nodes) of the server's trees.
        dict(name="append_16seq_8b", kind="append", n_seq=16, rows=25, take=5, ctx=4096, kv="f16",
             src="f32", **M8B),
        # A prompt's rows into a batch's caches.
        dict(name="append_64seq_8b", kind="append", n_seq=64, rows=150, take=150, ctx=512,
             kv="f16", src="f32", **M8B),
        # One user's decode step with a bounded cache.
        dict(name="scored_1seq_8b", kind="scored", n_seq=1, ctx=1000, kv="f16", **M8B),
        # A server's decode step over long ragged contexts.
        dict(name="scored_64seq_70b", kind="scored", n_seq=64, ctx=8192, kv="f16", **M70B),
        # A few sequences of a small model over fp32 caches.
        dict(name="scored_6seq_1b_f32", kind="scored", n_seq=6, ctx=3001, kv="f32", **M1B),
        # One user's cache brought back to its bound.
        dict(name="evict_1seq_8b", kind="evict", n_seq=1, ctx=1200, budget=512, kv="f16",
             place="in", **M8B),
        # A server's caches, in place.
        dict(name="evict_16seq_8b", kind="evict", n_seq=16, ctx=8192, budget=2048, kv="f16",
             place="in", **M8B),
        # Long prompts into the smaller caches they are decoded from.
        dict(name="evict_4seq_70b_long", kind="evict", n_seq=4, ctx=32768, budget=4000, kv="f16",
             place="out", **M70B),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["tree", "tree", "append", "scored", "scored", "evict"])
    if rng.random() < 0.5:
        w = dict(rng.choice([M8B, M70B, M1B]))
    else:
        n_kv = rng.choice([1, 2, 4, 8])
        w = {"n_heads": n_kv * rng.choice([1, 2, 4, 6, 8]), "n_kv": n_kv,
             "head_dim": rng.choice([64, 128])}
    kv = rng.choice(["f16", "f16", "f32"])
    n_seq = _log_int(rng, 1, 64)
    if kind == "append":
        rows = _log_int(rng, 1, 150)
        return dict(kind=kind, n_seq=n_seq, rows=rows, take=rng.randint(1, rows),
                    ctx=rows + _log_int(rng, 16, 350), kv=kv, src=rng.choice(["f32", "f16"]), **w)
    if kind == "scored":
        return dict(kind=kind, n_seq=n_seq, ctx=_log_int(rng, 16, 8192), kv=kv, **w)
    ctx = min(_log_int(rng, 16, 32768), 131072 // n_seq)
    if kind == "tree":
        return dict(kind=kind, n_seq=n_seq, nodes=_log_int(rng, 1, 64), ctx=ctx, kv=kv,
                    draft=rng.choice(["f32", "f16"]), **w)
    return dict(kind=kind, n_seq=n_seq, ctx=ctx, budget=max(8, int(ctx * rng.uniform(0.1, 0.9))),
                kv=kv, place=rng.choice(["in", "out"]), **w)


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------

def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed * 1000003 + 17)
    return g


def _randn(g, *shape, sigma=1.0, dtype=torch.float32):
    return torch.randn(*shape, generator=g, device="cuda").mul_(sigma).to(dtype)


def _type(name):
    return torch.float16 if name == "f16" else torch.float32


def _ints(a):
    return torch.from_numpy(np.ascontiguousarray(a, dtype=np.int32)).cuda()


def _lens(r, n, top):
    """Ragged lengths in [top / 2, top], the longest among them."""
    a = r.integers((top + 1) // 2, top + 1, size=n)
    a[0] = top
    return a


def _trees(r, n, T):
    """Parents of random trees [n, T] (-1: a child of the context's last token)
    and their ancestor masks, bit j of word j // 64."""
    parents = np.stack([r.integers(-1, i, size=n) if i else np.full(n, -1) for i in range(T)], 1)
    bits = np.zeros((n, T + 1, T), dtype=bool)  # row T: no ancestors
    for i in range(T):
        bits[:, i] = bits[np.arange(n), parents[:, i]]
        bits[:, i, i] = True
    words = (T + 63) // 64
    pad = np.zeros((n, T, words * 64), dtype=np.uint8)
    pad[:, :, :T] = bits[:, :T]
    return np.packbits(pad, axis=-1, bitorder="little").view(np.int64)


def _weights(g, n, nk, ctx):
    """Accumulated weights: heavy-tailed, on a grid coarse enough for ties."""
    w = torch.exp(torch.randn(n, nk, ctx, generator=g, device="cuda") * 2.0 - 4.0)
    return torch.round(w * 4096.0) / 4096.0


def prepare(case, seed):
    g, r = _gen(seed), np.random.default_rng(seed)
    n, ctx, nh, nk, hd = (case[k] for k in ("n_seq", "ctx", "n_heads", "n_kv", "head_dim"))
    kv, kind = _type(case["kv"]), case["kind"]
    s = {"case": case, "k": _randn(g, n, ctx, nk * hd, dtype=kv),
         "v": _randn(g, n, ctx, nk * hd, dtype=kv)}
    if kind == "tree":
        T, dt = case["nodes"], _type(case["draft"])
        s.update(q=_randn(g, n, T, nh * hd, sigma=2.0), k_draft=_randn(g, n, T, nk * hd, dtype=dt),
                 v_draft=_randn(g, n, T, nk * hd, dtype=dt), lens=_ints(_lens(r, n, ctx)),
                 mask=torch.from_numpy(_trees(r, n, T)).cuda(), n_nodes=_ints(_lens(r, n, T)),
                 out=torch.zeros(n, T, nh * hd, device="cuda"))
    elif kind == "append":
        R, A, dt = case["rows"], case["take"], _type(case["src"])
        index = np.sort(np.argsort(r.random((n, R)), axis=1)[:, :A], axis=1)
        s.update(k_rows=_randn(g, n, R, nk * hd, dtype=dt), v_rows=_randn(g, n, R, nk * hd, dtype=dt),
                 index=_ints(index), counts=_ints(r.integers(1, A + 1, size=n)),
                 lens=_ints(r.integers(0, ctx - A + 1, size=n)), weights=_weights(g, n, nk, ctx),
                 lens_out=torch.zeros(n, dtype=torch.int32, device="cuda"))
    elif kind == "scored":
        s.update(q=_randn(g, n, nh * hd, sigma=2.0), lens=_ints(_lens(r, n, ctx)),
                 weights=_weights(g, n, nk, ctx), out=torch.zeros(n, nh * hd, device="cuda"))
    else:
        B = case["budget"]
        s.update(weights=_weights(g, n, nk, ctx), lens=_ints(_lens(r, n, ctx)),
                 lens_out=torch.zeros(n, dtype=torch.int32, device="cuda"),
                 kept=torch.zeros(n, nk, B, dtype=torch.int32, device="cuda"))
        if case["place"] == "out":
            rows = B + 64  # room to decode on
            s.update(k_out=torch.zeros(n, rows, nk * hd, dtype=kv, device="cuda"),
                     v_out=torch.zeros(n, rows, nk * hd, dtype=kv, device="cuda"),
                     weights_out=torch.zeros(n, nk, rows, device="cuda"))
        else:
            s.update(k_out=s["k"], v_out=s["v"], weights_out=s["weights"])
    return s


def _protected(case):
    """The first and the most recent positions an eviction keeps."""
    return min(4, case["budget"] // 4), case["budget"] // 4


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------

def _heads(x, nk, hd):
    """[n, t, nk * hd] as fp32 [n, nk, t, hd]."""
    return x.float().reshape(x.shape[0], x.shape[1], nk, hd).permute(0, 2, 1, 3)


def _softmax(z, live):
    """exp(z - max) over the live columns and its row sums."""
    z = torch.where(live, z, torch.full_like(z, -math.inf))
    m = z.amax(-1, keepdim=True)
    p = torch.exp(z - torch.where(m > -math.inf, m, torch.zeros_like(m)))
    return p, p.sum(-1, keepdim=True)


def _plain_tree(s):
    c = s["case"]
    n, ctx, T, nh, nk, hd = (c[k] for k in ("n_seq", "ctx", "nodes", "n_heads", "n_kv", "head_dim"))
    g = nh // nk
    k = torch.cat((s["k"], s["k_draft"].to(s["k"].dtype)), 1)
    v = torch.cat((s["v"], s["v_draft"].to(s["v"].dtype)), 1)
    q = s["q"].reshape(n, T, nk, g, hd).permute(0, 2, 1, 3, 4).reshape(n, nk, T * g, hd)
    z = (q @ _heads(k, nk, hd).transpose(-1, -2).contiguous()) * (1.0 / math.sqrt(hd))
    at = torch.arange(T, device="cuda")
    near = ((s["mask"][:, :, at // 64] >> (at % 64)) & 1).bool()
    near = near & (at < s["n_nodes"][:, None])[:, None, :]
    far = torch.arange(ctx, device="cuda") < s["lens"][:, None]
    live = torch.cat((far[:, None, :].expand(n, T, ctx), near), -1)
    p, total = _softmax(z, live[:, None, :, None, :].expand(n, 1, T, g, ctx + T)
                        .reshape(n, 1, T * g, ctx + T))
    o = (p @ _heads(v, nk, hd).contiguous()) / torch.where(total > 0, total, torch.ones_like(total))
    o = o.reshape(n, nk, T, g, hd).permute(0, 2, 1, 3, 4).reshape(n, T, nh * hd)
    s["out"].copy_(torch.where((at < s["n_nodes"][:, None])[:, :, None], o, s["out"]))
    return s["out"]


def _plain_scored(s):
    c = s["case"]
    n, ctx, nh, nk, hd = (c[k] for k in ("n_seq", "ctx", "n_heads", "n_kv", "head_dim"))
    q = s["q"].reshape(n, nk, nh // nk, hd)
    z = (q @ _heads(s["k"], nk, hd).transpose(-1, -2).contiguous()) * (1.0 / math.sqrt(hd))
    live = (torch.arange(ctx, device="cuda") < s["lens"][:, None])[:, None, None, :]
    p, total = _softmax(z, live)
    s["out"].copy_(((p @ _heads(s["v"], nk, hd).contiguous()) / total).reshape(n, nh * hd))
    s["weights"].add_((p / total).sum(2))
    return s["out"], s["weights"]


def _plain_append(s):
    c = s["case"]
    n, A, ctx = c["n_seq"], c["take"], c["ctx"]
    a = torch.arange(A, device="cuda")
    seq, j = torch.nonzero(a < s["counts"][:, None], as_tuple=True)
    pos, row = s["lens"][seq].long() + j, s["index"][seq, j].long()
    s["k"][seq, pos] = s["k_rows"][seq, row].to(s["k"].dtype)
    s["v"][seq, pos] = s["v_rows"][seq, row].to(s["v"].dtype)
    s["weights"].transpose(1, 2)[seq, pos] = 0.0
    s["lens_out"].copy_(s["lens"] + s["counts"])
    return s["k"], s["v"], s["weights"], s["lens_out"]


def _plain_evict(s):
    c = s["case"]
    n, ctx, nk, hd, B = (c[k] for k in ("n_seq", "ctx", "n_kv", "head_dim", "budget"))
    first, recent = _protected(c)
    t = torch.arange(ctx, device="cuda")
    ln = s["lens"][:, None, None]
    w = torch.where((t < first) | (t >= ln - recent), math.inf, s["weights"])
    w = torch.where(t < ln, w, -math.inf)
    B = min(B, ctx)
    at = torch.sort(w, dim=-1, descending=True, stable=True).indices[..., :B].sort(-1).values
    live = torch.arange(B, device="cuda") < torch.minimum(s["lens"], torch.full_like(s["lens"], B))[:, None]
    s["kept"].fill_(-1)
    s["kept"][..., :B] = torch.where(live[:, None], at, -1).int()
    rows = at.transpose(1, 2)[..., None].expand(n, B, nk, hd)
    for name in ("k", "v"):
        new = torch.gather(s[name].reshape(n, ctx, nk, hd), 1, rows).reshape(n, B, nk * hd)
        out = s[name + "_out"][:, :B]
        out.copy_(torch.where(live[:, :, None], new, out))
    out = s["weights_out"][..., :B]
    out.copy_(torch.where(live[:, None], torch.gather(s["weights"], 2, at), out))
    s["lens_out"].copy_(torch.minimum(s["lens"], torch.full_like(s["lens"], B)))
    return s["k_out"], s["v_out"], s["weights_out"], s["kept"], s["lens_out"]


def _jinf():
    path = os.path.abspath("jetson-inference_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import jinf_amd

    return jinf_amd


def _workspace(s, make, *args):
    """The call's workspace, made by the first pass and kept as a user's program keeps it."""
    if "workspace" not in s:
        s["workspace"] = make(*args)
    return s["workspace"]


def run(state):
    s, c = state, state["case"]
    kind = c["kind"]
    if not own:
        return {"tree": _plain_tree, "append": _plain_append, "scored": _plain_scored,
                "evict": _plain_evict}[kind](s)
    jinf = _jinf()
    n, ctx, nh, nk, hd = (c[k] for k in ("n_seq", "ctx", "n_heads", "n_kv", "head_dim"))
    if kind == "tree":
        ws = _workspace(s, jinf.attention_tree_workspace, n, c["nodes"], nh, nk, hd, ctx)
        return jinf.attention_tree(s["q"], s["k"], s["v"], s["lens"], s["k_draft"], s["v_draft"],
                                   s["mask"], nh, nk, n_nodes=s["n_nodes"], out=s["out"],
                                   workspace=ws)
    if kind == "append":
        lens = jinf.cache_append(s["k"], s["v"], s["lens"], s["k_rows"], s["v_rows"], nk,
                                 index=s["index"], counts=s["counts"], weights=s["weights"],
                                 lens_out=s["lens_out"])
        return s["k"], s["v"], s["weights"], lens
    if kind == "scored":
        ws = _workspace(s, jinf.attention_scored_workspace, n, nh, nk, hd, ctx)
        out = jinf.attention_decode_scored(s["q"], s["k"], s["v"], s["lens"], s["weights"], nh, nk,
                                           out=s["out"], workspace=ws)
        return out, s["weights"]
    first, recent = _protected(c)
    ws = _workspace(s, jinf.cache_evict_workspace, n, nk, c["budget"])
    lens = jinf.cache_evict(s["k"], s["v"], s["weights"], s["lens"], nk, c["budget"],
                            n_first=first, n_recent=recent, k_out=s["k_out"], v_out=s["v_out"],
                            weights_out=s["weights_out"], lens_out=s["lens_out"], kept=s["kept"],
                            workspace=ws)
    return s["k_out"], s["v_out"], s["weights_out"], s["kept"], lens


def work(case):
    n, ctx, nh, nk, hd = (case[k] for k in ("n_seq", "ctx", "n_heads", "n_kv", "head_dim"))
    es, kvw = (2 if case["kv"] == "f16" else 4), nk * hd
    mean = (ctx + (n - 1) * 0.75 * ctx) / n  # of the ragged lengths
    if case["kind"] == "append":
        live, ss = n * (case["take"] + 1) / 2, (2 if case["src"] == "f16" else 4)
        return {"bytes": live * (2 * kvw * (es + ss) + 4 * nk) + 12 * n, "flops": 0}
    if case["kind"] == "evict":
        rows = n * min(case["budget"], mean)
        return {"bytes": n * nk * mean * 4 + rows * (4 * kvw * es + 12 * nk), "flops": 0}
    if case["kind"] == "tree":
        ds = 2 if case["draft"] == "f16" else 4
        T = case["nodes"]
        live = n * (T + (n - 1) * 0.75 * T) / n
        return {"bytes": 2 * kvw * (n * mean * es + live * ds) + live * nh * hd * 8
                + live * 8 * ((T + 63) // 64),
                "flops": 4 * hd * nh * live * (mean + 1 + math.log(T))}
    return {"bytes": n * mean * (2 * kvw * es + 8 * nk) + n * nh * hd * 8,
            "flops": 4 * hd * nh * n * mean}


# ---------------------------------------------------------------------------
# 64 bits
# ---------------------------------------------------------------------------

def _attend(q, k, v, seen):
    """q [rows, hd] over k, v [t, hd] where seen [rows, t]: outputs and weights."""
    z = (q.double() @ k.double().t().contiguous()) / math.sqrt(q.shape[1])
    z.masked_fill_(~seen, -math.inf)
    p = torch.softmax(z, -1)
    p[~seen.any(-1)] = 0.0
    return p @ v.double(), p


def exact(case, seed):
    s = prepare(case, seed)
    n, ctx, nh, nk, hd = (case[k] for k in ("n_seq", "ctx", "n_heads", "n_kv", "head_dim"))
    g, kind = nh // nk, case["kind"]
    lens = s["lens"].tolist()
    if kind == "append":
        k, v, w = s["k"].double(), s["v"].double(), s["weights"].double()
        for i in range(n):
            for a in range(int(s["counts"][i])):
                row, t = int(s["index"][i, a]), lens[i] + a
                k[i, t] = s["k_rows"][i, row].to(s["k"].dtype).double()
                v[i, t] = s["v_rows"][i, row].to(s["v"].dtype).double()
                w[i, :, t] = 0.0
        return k, v, w, None
    if kind == "evict":
        first, recent = _protected(case)
        k, v, w = (s[x].double() for x in ("k_out", "v_out", "weights_out"))
        for i in range(n):
            for j in range(nk):
                m = min(case["budget"], lens[i])
                mid = s["weights"][i, j, first:lens[i] - recent].double().cpu().numpy()
                keep = list(range(lens[i]))
                if lens[i] > m:
                    best = np.lexsort((np.arange(mid.size), -mid))[:m - first - recent]
                    keep = list(range(first)) + sorted(int(b) + first for b in best)
                    keep += list(range(lens[i] - recent, lens[i]))
                keep = torch.tensor(keep, device="cuda", dtype=torch.long)
                cols = slice(j * hd, (j + 1) * hd)
                k[i, :m, cols] = s["k"][i, keep, cols].double()
                v[i, :m, cols] = s["v"][i, keep, cols].double()
                w[i, j, :m] = s["weights"][i, j, keep].double()
        return k, v, w, None, None
    out = s["out"].double()
    if kind == "scored":
        w = s["weights"].double()
        for i, t in enumerate(lens):
            for j in range(nk):
                q = s["q"][i].reshape(nh, hd)[j * g:(j + 1) * g]
                cols = slice(j * hd, (j + 1) * hd)
                o, p = _attend(q, s["k"][i, :t, cols], s["v"][i, :t, cols],
                               torch.ones(g, t, dtype=torch.bool, device="cuda"))
                out[i, j * g * hd:(j + 1) * g * hd] = o.reshape(-1)
                w[i, j, :t] += p.sum(0)
        return out, w
    for i, t in enumerate(lens):
        m = int(s["n_nodes"][i])
        words = s["mask"][i, :m].cpu().numpy().view(np.uint8).reshape(m, -1)
        near = torch.from_numpy(np.unpackbits(words, axis=1, bitorder="little")[:, :m]).cuda().bool()
        seen = torch.cat((torch.ones(m, t, dtype=torch.bool, device="cuda"), near), 1)
        seen = seen.repeat_interleave(g, 0)
        for j in range(nk):
            cols = slice(j * hd, (j + 1) * hd)
            k, v = (torch.cat((s[x][i, :t, cols], s[x + "_draft"][i, :m, cols].to(s[x].dtype)))
                    for x in ("k", "v"))
            q = s["q"][i, :m].reshape(m, nh, hd)[:, j * g:(j + 1) * g].reshape(m * g, hd)
            o, _ = _attend(q, k, v, seen)
            out.view(n, -1, nh, hd)[i, :m, j * g:(j + 1) * g] = o.reshape(m, g, hd)
    return out
