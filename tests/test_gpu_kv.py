"""GPU: attention of drafted tokens, cache appends, decode attention with summed
weights and cache eviction, against the 64-bit forms of kv_ref.py.

Bars.  Attention outputs: |err| <= 2e-5 sum p |v|, the bar of the decode
attention (an exponential within 6.5e-6 over the whole range of normal results,
a score of about 22 bits).  Summed weights: each step's weight within 2e-5 of
itself and one fp32 addition, half a step of the sum (2^-24).  Everything the
append and the eviction store is a copy or one rounding: equal bits.

What must not be read is NaN: cache positions past a length, drafted rows past a
sequence's nodes.
"""
import numpy as np
import pytest
import torch

import jinf_amd
import kv_ref
from gpu_util import host, say
from jinf_amd import JinfError

pytestmark = pytest.mark.gpu

DT = {"f16": torch.float16, "f32": torch.float32}
NAN = float("nan")


def rand(seed, *shape, sigma=1.0, dtype=torch.float32):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * sigma).to(dtype)


def strided(t, pad, fill=NAN):
    """t on the device with `pad` more elements between its last-but-one rows."""
    big = torch.full((*t.shape[:-1], t.shape[-1] + pad), fill, dtype=t.dtype, device="cuda")
    big[..., :t.shape[-1]] = t.cuda()
    return big[..., :t.shape[-1]]


def ints(a):
    return torch.tensor(np.asarray(a), dtype=torch.int32, device="cuda")


def caches(seed, n, ctx, kvw, dt, lens, pad=0):
    """K / V on the host, and on the device with NaN past each length."""
    out = []
    for x in range(2):
        t = rand(seed + x, n, ctx, kvw, dtype=dt)
        d = strided(t, pad)
        for s in range(n):
            d[s, max(int(lens[s]), 0):] = NAN
        out += [t, d]
    return out[0], out[2], out[1], out[3]


def close(got, want, mag, what, bar=2e-5):
    err = np.abs(got.astype(np.float64) - want)
    bad = ~(err <= bar * mag + 1e-30)
    worst = float(np.nanmax(err / np.maximum(mag, 1e-30))) if err.size else 0.0
    say(f"{what}: worst error / sum p|v| = {worst:.2e}")
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.size} off, worst {worst:.2e}"


def random_mask(r, n, T, density=None):
    """A tree's mask, or any relation of this density."""
    if density is None:
        par = np.stack([r.integers(-1, i, size=n) if i else np.full(n, -1) for i in range(T)], 1)
        return jinf_amd.tree_mask(par)
    words = (T + 63) // 64
    bits = np.zeros((n, T, words * 64), np.uint8)
    bits[:, :, :T] = r.random((n, T, T)) < density
    return torch.from_numpy(np.packbits(bits, -1, bitorder="little").view(np.int64).copy()).cuda()


def run_tree(n, T, ctx, nh, nk, hd, kv, draft, lens, n_nodes=None, density=None, pad=0, sigma=2.0,
             split=True, wide=False):
    r = np.random.default_rng(n * 7919 + T * 31 + ctx)
    dt = DT[kv]
    k, v, kg, vg = caches(T + ctx, n, ctx, nk * hd, dt, lens, pad)
    q = rand(3 + T, n, T, nh * hd, sigma=sigma)
    kd = rand(5 + T, n, T, nk * hd, dtype=DT[draft])
    vd = rand(6 + T, n, T, nk * hd, dtype=DT[draft])
    mask = random_mask(r, n, T, density)
    qg, kdg, vdg = strided(q, pad), strided(kd, pad), strided(vd, pad)
    if n_nodes is not None:
        for s in range(n):
            for t in (qg, kdg, vdg):
                t[s, max(n_nodes[s], 0):] = NAN
    out = strided(torch.full((n, T, nh * hd), -3.0), pad, -3.0)
    ws = None if split else torch.empty(16, dtype=torch.uint8, device="cuda")
    got = jinf_amd.attention_tree(qg, kg, vg, ints(lens), kdg, vdg, mask, nh, nk,
                                  n_nodes=None if n_nodes is None else ints(n_nodes), out=out,
                                  workspace=ws)
    assert got is out
    want, mag = kv_ref.tree(q, k, v, lens, kd, vd, mask, nh, nk, n_nodes)
    got = host(got)
    bar = 2e-5
    if wide:
        # Scores far from 0.  An fp32 sum of hd products in any order is off by at
        # most hd 2^-24 of the sum A of their magnitudes, the scaled and split q
        # by another 4 2^-24 A: each score by d = (hd + 4) 2^-24 A at most, so
        # each exponential by a factor within e^(+-d), each probability (an
        # exponential over a sum of them) within e^(+-2 d), and the output by
        # (e^(2 d) - 1) sum p |v|.
        A = 0.0
        for j in range(nk):
            c = slice(j * hd, (j + 1) * hd)
            keys = torch.cat((k[..., c], kd.to(dt)[..., c]), 1).double().abs()
            qs = q.double().reshape(n, T, nk, nh // nk, hd)[:, :, j].reshape(n, -1, hd).abs()
            A = max(A, float((qs @ keys.transpose(1, 2)).max()) / np.sqrt(hd))
        bar += np.expm1(2 * (hd + 4) * 2.0 ** -24 * A)
    for s in range(n):
        m = T if n_nodes is None else min(max(n_nodes[s], 0), T)
        assert np.all(got[s, m:] == -3.0), "rows past the nodes were written"
        close(got[s, :m], want[s, :m], mag[s, :m],
              f"tree n={n} T={T} ctx={ctx} {nh}/{nk}x{hd} {kv}/{draft} seq {s} len {lens[s]} nodes {m}", bar)
    return got


@pytest.mark.parametrize("kv,draft", [("f16", "f32"), ("f16", "f16"), ("f32", "f32"), ("f32", "f16")])
@pytest.mark.parametrize("n,T,ctx,nh,nk,hd", [
    (1, 1, 1, 1, 1, 64), (1, 1, 65, 8, 8, 128), (2, 7, 333, 32, 8, 128), (3, 13, 200, 32, 8, 64),
    (2, 25, 1111, 12, 2, 128), (1, 64, 700, 16, 2, 64), (2, 65, 130, 4, 4, 64),
    (1, 130, 257, 8, 1, 128), (1, 256, 90, 4, 2, 128), (4, 3, 64, 28, 4, 128), (1, 5, 500, 40, 1, 64),
])
def test_tree_shapes(dev, n, T, ctx, nh, nk, hd, kv, draft):
    r = np.random.default_rng(ctx)
    lens = [ctx] + [int(x) for x in r.integers(0, ctx + 1, size=n - 1)]
    run_tree(n, T, ctx, nh, nk, hd, kv, draft, lens)


@pytest.mark.parametrize("kv", list(DT))
@pytest.mark.parametrize("hd,pad", [(80, 0), (96, 3), (1, 0), (256, 0), (64, 1), (128, 8), (128, 4)])
def test_tree_other_layouts(dev, hd, pad, kv):
    """Head sizes and strides off the fast path, and on it with gaps between rows."""
    run_tree(2, 6, 77, 4, 2, hd, kv, "f32", [77, 20], pad=pad)


@pytest.mark.parametrize("kv", list(DT))
@pytest.mark.parametrize("hd", [64, 128, 96])
def test_tree_lengths_and_node_counts(dev, kv, hd):
    """Empty contexts, lengths past either bound, sequences of fewer nodes, none at
    all, or more than there are."""
    run_tree(7, 10, 300, 8, 2, hd, kv, "f32", [0, 1, 63, 64, -5, 999, 300],
             n_nodes=[10, 1, 0, 7, 3, -2, 99])


@pytest.mark.parametrize("kv", list(DT))
@pytest.mark.parametrize("density", [0.0, 0.03, 0.5, 1.0])
def test_tree_any_relation(dev, kv, density):
    """Masks that are no trees: rows that see nothing give zeros where the context
    is empty, and the context alone elsewhere."""
    got = run_tree(3, 70, 100, 8, 2, 64, kv, "f32", [0, 100, 3], density=density)
    if density == 0.0:
        assert np.all(got[0] == 0.0)


@pytest.mark.parametrize("kv", list(DT))
@pytest.mark.parametrize("T", [2, 33, 64])
def test_tree_split_and_whole_contexts(dev, kv, T):
    """Long ragged contexts, with the workspace that splits them and without."""
    for split in (True, False):
        run_tree(3, T, 5000, 8, 2, 128, kv, "f32", [5000, 259, 4100], split=split)


def test_tree_shared_prefix(dev):
    """Every sequence over one cached prefix (sequence stride 0)."""
    k, v = rand(1, 1, 400, 256, dtype=torch.float16), rand(2, 1, 400, 256, dtype=torch.float16)
    q, kd, vd = rand(3, 4, 6, 1024), rand(4, 4, 6, 256), rand(5, 4, 6, 256)
    lens, mask = [400, 399, 7, 200], random_mask(np.random.default_rng(1), 4, 6)
    kg, vg = k.cuda().expand(4, -1, -1), v.cuda().expand(4, -1, -1)
    got = jinf_amd.attention_tree(q.cuda(), kg, vg, ints(lens), kd.cuda(), vd.cuda(), mask, 8, 2)
    want, mag = kv_ref.tree(q, k.expand(4, -1, -1), v.expand(4, -1, -1), lens, kd, vd, mask, 8, 2)
    close(host(got), want, mag, "shared prefix")


@pytest.mark.parametrize("kv", list(DT))
@pytest.mark.parametrize("hd", [64, 128, 32])
def test_tree_non_finite_values(dev, kv, hd):
    """Infinities and NaN in drafted rows stay with the nodes that see them: a NaN
    key makes those nodes NaN, a non-finite value its dim in them; the others are
    as without it.  A NaN in q stays in its node and head."""
    n, T, ctx, nh, nk = 1, 20, 150, 8, 2
    r = np.random.default_rng(hd)
    k, v, kg, vg = caches(1, n, ctx, nk * hd, DT[kv], [ctx])
    q, kd, vd = rand(3, n, T, nh * hd), rand(4, n, T, nk * hd), rand(5, n, T, nk * hd)
    mask = random_mask(r, n, T, 0.3)
    bits = kv_ref.mask_bits(mask)[0]
    want, mag = kv_ref.tree(q, k, v, [ctx], kd, vd, mask, nh, nk)
    nan = np.zeros(want.shape, bool).reshape(n, T, nh, hd)
    g = nh // nk
    kd[0, 3, :hd] = NAN                       # node 3's key, kv head 0
    nan[0, bits[:, 3], :g] = True
    for node, j, d, x in ((5, 1, 2, np.inf), (11, 0, hd - 1, -np.inf), (19, 1, 7, NAN)):
        vd[0, node, j * hd + d] = x
        nan[0, bits[:, node], j * g:(j + 1) * g, d] = True
    q[0, 8, hd:hd + 3] = NAN                  # node 8, head 1
    nan[0, 8, 1] = True
    nan = nan.reshape(want.shape)
    got = host(jinf_amd.attention_tree(q.cuda(), kg, vg, ints([ctx]), kd.cuda(), vd.cuda(), mask,
                                       nh, nk))
    inf = np.isinf(got)  # an infinite value may stay one in the dims it makes non-finite
    assert np.array_equal(np.isnan(got) | inf, nan)
    close(got[~nan], want[~nan], mag[~nan], "finite places")


def test_tree_scores_of_any_size(dev):
    """Scores far apart, and all equal to the lowest fp16 value's products."""
    run_tree(1, 9, 300, 4, 2, 64, "f16", "f32", [300], sigma=200.0, wide=True)
    run_tree(1, 9, 300, 4, 2, 64, "f32", "f32", [300], sigma=200.0, wide=True)
    n, T, ctx, hd = 1, 3, 70, 64
    k = torch.full((n, ctx, hd), -65504.0, dtype=torch.float16)
    v = rand(2, n, ctx, hd, dtype=torch.float16)
    q, kd, vd = torch.ones(n, T, hd), torch.full((n, T, hd), -65504.0), rand(3, n, T, hd)
    mask = jinf_amd.tree_mask([[-1, 0, 0]])
    got = jinf_amd.attention_tree(q.cuda(), k.cuda(), v.cuda(), ints([ctx]), kd.cuda(), vd.cuda(),
                                  mask, 1, 1)
    want, mag = kv_ref.tree(q, k, v, [ctx], kd, vd, mask, 1, 1)
    close(host(got), want, mag, "lowest scores")


def test_tree_cache_past_32_bit_offsets(dev):
    """A cache whose positions lie more than 2^32 bytes apart in all."""
    ctx, kvw, ld = 1500, 128, 2_000_000
    big = torch.empty(ctx * ld + kvw, dtype=torch.float16, device="cuda")
    k, v = rand(1, 1, ctx, kvw, dtype=torch.float16), rand(2, 1, ctx, kvw, dtype=torch.float16)
    kg, vg = (big.as_strided((1, ctx, kvw), (ctx * ld, ld, 1), o) for o in (0, 1024))
    kg.copy_(k), vg.copy_(v)
    q, kd, vd = rand(3, 1, 5, 256), rand(4, 1, 5, kvw), rand(5, 1, 5, kvw)
    mask = random_mask(np.random.default_rng(1), 1, 5)
    got = jinf_amd.attention_tree(q.cuda(), kg, vg, ints([ctx]), kd.cuda(), vd.cuda(), mask, 4, 2)
    want, mag = kv_ref.tree(q, k, v, [ctx], kd, vd, mask, 4, 2)
    close(host(got), want, mag, "far positions")
    w = torch.zeros(1, 2, ctx, device="cuda")
    got = jinf_amd.attention_decode_scored(q[:, 0].cuda(), kg, vg, ints([ctx]), w, 4, 2)
    want, mag, ww = kv_ref.scored(q[:, 0], k, v, [ctx], 4, 2)
    close(host(got), want, mag, "far positions, one token")
    close(host(w), ww, ww, "far positions' weights")


@pytest.mark.parametrize("kv,ctx", [("f16", 17000), ("f32", 8500)])
@pytest.mark.parametrize("T", [3, 10, 25, 50])
def test_tree_large_caches(dev, kv, ctx, T):
    """Caches past 128 MB, which take loads and tile counts of their own, at each number
    of rows a workgroup holds (6 to 100 rows a kv head)."""
    run_tree(2, T, ctx, 16, 8, 128, kv, "f32", [ctx, ctx // 2 + 1], n_nodes=[T, max(1, T // 2)])


def test_tree_large_caches_of_narrow_heads(dev):
    run_tree(2, 7, 17000, 32, 16, 64, "f16", "f16", [17000, 63])


@pytest.mark.parametrize("n,T,ctx,nh,kv,lens,n_nodes", [
    (5, 20, 14000, 16, "f16", [14000, 0, 1, 137, 9000], [20, 20, 0, 7, 13]),
    (5, 20, 14000, 16, "f16", [40, 0, 0, 0, 0], [20, 3, 1, 0, 20]),
    (5, 20, 14000, 16, "f16", [0, 14000, 14000, 14000, 14000], [0, 20, 20, 20, 20]),
    (2, 256, 33000, 8, "f16", [300, 10000], [256, 70]),
    (3, 20, 24000, 16, "f32", [24000, 640, 5], None),
    (8, 3, 33000, 16, "f16", [33000, 0, 5, 12000, 700, 64, 2000, 1], [3, 3, 1, 2, 0, 3, 1, 3]),
])
def test_tree_ragged_work_in_equal_shares(dev, n, T, ctx, nh, kv, lens, n_nodes):
    """Caches much longer than most contexts, sequences of many and no nodes: work that
    the kernel divides by the lengths and counts it finds."""
    run_tree(n, T, ctx, nh, 8, 64, kv, "f32", lens, n_nodes=n_nodes)


def test_tree_shares_follow_the_lengths_of_each_replay(dev):
    """One captured call, replayed as lengths and node counts change."""
    n, T, ctx, nh, nk, hd = 5, 20, 14000, 16, 8, 64
    k, v = (rand(i, n, ctx, nk * hd, dtype=torch.float16).cuda() for i in (1, 2))
    q, kd, vd = rand(3, n, T, nh * hd).cuda(), rand(4, n, T, nk * hd).cuda(), rand(5, n, T, nk * hd).cuda()
    mask = random_mask(np.random.default_rng(7), n, T)
    lens, nodes = ints([14000] * n), ints([T] * n)
    ws = jinf_amd.attention_tree_workspace(n, T, nh, nk, hd, ctx)
    out = torch.zeros(n, T, nh * hd, device=dev)
    args = (q, k, v, lens, kd, vd, mask, nh, nk, nodes)
    jinf_amd.attention_tree(*args, out=out, workspace=ws)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        jinf_amd.attention_tree(*args, out=out, workspace=ws)
    for step, (a, b) in enumerate([([14000] * 5, [20] * 5), ([1, 14000, 0, 333, 7000], [20, 1, 5, 0, 19]),
                                   ([0] * 5, [0, 0, 0, 0, 20]), ([9000, 9001, 64, 63, 2], [3] * 5)]):
        lens.copy_(ints(a)), nodes.copy_(ints(b))
        out.fill_(-3.0)
        torch.cuda.synchronize()
        g.replay()
        got = host(out).copy()
        torch.cuda.synchronize()
        say(f"replay {step} of lengths {a}, nodes {b}")
        want = torch.full_like(out, -3.0)
        jinf_amd.attention_tree(*args, out=want, workspace=ws.clone())
        assert np.array_equal(got, host(want)), step
        whole = torch.full_like(out, -3.0)  # every context in one piece
        jinf_amd.attention_tree(*args, out=whole, workspace=torch.empty(16, dtype=torch.uint8, device=dev))
        top = v.float().abs().max().item()  # both within 2e-5 sum p |v| of the exact result
        assert np.all(np.abs(got - host(whole)) <= 4e-5 * max(top, vd.abs().max().item())), step


def test_one_workspace_for_calls_of_many_shapes(dev):
    """A workspace of the largest shape serves smaller ones in any order, whatever it
    held before; two calls on two streams, with one each, do not disturb each other."""
    shapes = [(3, 30, 3000, 8, 2), (1, 3, 2999, 8, 2), (2, 64, 1500, 8, 2), (3, 1, 640, 8, 2)]
    size = max(jinf_amd.attention_tree_workspace(n, T, nh, nk, 64, ctx).numel()
               for n, T, ctx, nh, nk in shapes)
    top = jinf_amd.attention_tree_workspace(3, 64, 8, 2, 64, 3000)
    assert top.numel() >= size
    top.fill_(255)
    calls = []
    for n, T, ctx, nh, nk in shapes:
        k, v = (rand(i, n, ctx, nk * 64, dtype=torch.float16) for i in (1, 2))
        q, kd, vd = rand(3, n, T, nh * 64), rand(4, n, T, nk * 64), rand(5, n, T, nk * 64)
        mask = random_mask(np.random.default_rng(T), n, T)
        lens = [ctx] * n
        args = (q.cuda(), k.cuda(), v.cuda(), ints(lens), kd.cuda(), vd.cuda(), mask, nh, nk)
        got = host(jinf_amd.attention_tree(*args, workspace=top)).copy()
        want, mag = kv_ref.tree(q, k, v, lens, kd, vd, mask, nh, nk)
        close(got, want, mag, f"shared workspace n={n} T={T} ctx={ctx}")
        calls.append((args, got))
    streams, outs = [torch.cuda.Stream() for _ in calls], []
    spaces = [jinf_amd.attention_tree_workspace(n, T, nh, nk, 64, ctx) for n, T, ctx, nh, nk in shapes]
    torch.cuda.synchronize()
    for (args, _), st, ws in zip(calls, streams, spaces):
        with torch.cuda.stream(st):
            outs.append(jinf_amd.attention_tree(*args, workspace=ws))
    torch.cuda.synchronize()
    for (_, got), out in zip(calls, outs):
        assert np.array_equal(host(out), got)


# ---- one token with summed weights ----

def run_scored(n, ctx, nh, nk, hd, kv, lens, pad=0, steps=2):
    dt = DT[kv]
    k, v, kg, vg = caches(ctx, n, ctx, nk * hd, dt, lens, pad)
    w0 = rand(9, n, nk, ctx).abs()
    wg = strided(w0, pad, -1.0)
    want_w = w0.double().numpy()
    ws = jinf_amd.attention_scored_workspace(n, nh, nk, hd, ctx)
    for step in range(steps):
        q = rand(30 + step, n, nh * hd, sigma=2.0)
        out = strided(torch.full((n, nh * hd), -3.0), pad, -3.0)
        jinf_amd.attention_decode_scored(strided(q, pad), kg, vg, ints(lens), wg, nh, nk, out=out,
                                         workspace=ws)
        want, mag, w = kv_ref.scored(q, k, v, lens, nh, nk)
        what = f"scored n={n} ctx={ctx} {nh}/{nk}x{hd} {kv} step {step}"
        close(host(out), want, mag, what)
        prev = host(wg) if step else w0.numpy()
        want_w = want_w + w
        bar = (step + 1) * 2.0 ** -24 * want_w + 2e-5 * (want_w - w0.double().numpy()) + 1e-30
        got = host(wg)
        assert np.all(np.abs(got - want_w) <= bar), what
        for s in range(n):
            t = min(max(int(lens[s]), 0), ctx)
            assert np.array_equal(got[s, :, t:], w0.numpy()[s, :, t:]), "weights past the length"
        del prev


@pytest.mark.parametrize("kv", list(DT))
@pytest.mark.parametrize("n,ctx,nh,nk,hd", [
    (1, 1, 1, 1, 64), (1, 1000, 32, 8, 128), (6, 777, 32, 8, 64), (3, 4097, 64, 8, 128),
    (2, 300, 12, 2, 128), (2, 130, 6, 6, 64), (1, 9000, 40, 1, 128), (5, 64, 28, 4, 128),
    (3, 90, 4, 2, 80), (2, 90, 4, 2, 256),
])
def test_scored_shapes(dev, n, ctx, nh, nk, hd, kv):
    r = np.random.default_rng(ctx)
    run_scored(n, ctx, nh, nk, hd, kv, [ctx] + [int(x) for x in r.integers(0, ctx + 1, size=n - 1)])


@pytest.mark.parametrize("kv", list(DT))
@pytest.mark.parametrize("pad", [1, 8])
def test_scored_lengths_and_strides(dev, kv, pad):
    run_scored(6, 200, 8, 2, 64, kv, [0, 1, 64, 65, -3, 500], pad=pad)


@pytest.mark.parametrize("kv,ctx,nh,nk,hd", [("f16", 17000, 16, 8, 128), ("f32", 8500, 16, 8, 128),
                                             ("f16", 17000, 160, 8, 128), ("f16", 17000, 64, 16, 64)])
def test_scored_large_caches(dev, kv, ctx, nh, nk, hd):
    """Caches past 128 MB, 2, 4 and 20 query heads a kv head."""
    run_scored(2, ctx, nh, nk, hd, kv, [ctx, 4321], steps=1)


@pytest.mark.parametrize("lens", [[33000, 0, 5, 12000, 700, 64, 2000, 1], [0] * 7 + [130]])
def test_scored_ragged_work_in_equal_shares(dev, lens):
    run_scored(8, 33000, 16, 8, 64, "f16", lens, steps=1)


@pytest.mark.parametrize("kv", list(DT))
def test_scored_matches_the_decode_attention(dev, kv):
    """The output is the decode attention's, within twice the bar both keep."""
    n, ctx, nh, nk, hd = 4, 1500, 32, 8, 128
    k, v = (rand(i, n, ctx, nk * hd, dtype=DT[kv]).cuda() for i in (1, 2))
    q, lens = rand(3, n, nh * hd).cuda(), ints([1500, 3, 800, 257])
    a = host(jinf_amd.attention_decode(q, k, v, lens, nh, nk))
    b = host(jinf_amd.attention_decode_scored(q, k, v, lens, torch.zeros(n, nk, ctx, device=dev),
                                              nh, nk))
    _, mag, _ = kv_ref.scored(q, k, v, lens, nh, nk)
    assert np.all(np.abs(a.astype(np.float64) - b) <= 4e-5 * mag)


def test_scored_nan_stays_in_its_kv_head(dev):
    n, ctx, nh, nk, hd = 1, 300, 8, 2, 128
    k, v = (rand(i, n, ctx, nk * hd, dtype=torch.float16).cuda() for i in (1, 2))
    k[0, 100, :hd] = NAN
    w = torch.zeros(n, nk, ctx, device=dev)
    out = host(jinf_amd.attention_decode_scored(rand(3, n, nh * hd).cuda(), k, v, ints([ctx]), w, nh,
                                                nk)).reshape(nh, hd)
    w = host(w)
    assert np.isnan(out[:4]).all() and np.isfinite(out[4:]).all()
    assert np.isnan(w[0, 0]).all() and np.isfinite(w[0, 1]).all()


# ---- appends ----

@pytest.mark.parametrize("kv", list(DT))
@pytest.mark.parametrize("src", list(DT))
@pytest.mark.parametrize("nk,hd,pad", [(2, 64, 0), (8, 128, 8), (3, 20, 1), (1, 1, 0)])
def test_append(dev, kv, src, nk, hd, pad):
    """Ragged counts past both bounds, rows named twice and outside the rows, and
    positions past the cache's end."""
    n, ctx, rows, take, kvw = 5, 40, 9, 6, nk * hd
    k, v = (strided(rand(i, n, ctx, kvw, dtype=DT[kv]), pad) for i in (1, 2))
    kr, vr = (rand(i, n, rows, kvw, sigma=3.0, dtype=DT[src]) for i in (3, 4))
    w = strided(rand(5, n, nk, ctx).abs() + 1.0, pad)
    index = np.array([[8, 8, 0, 1, 2, 3], [-1, 9, 4, 5, 6, 7], [0, 1, 2, 3, 4, 5],
                      [5, 4, 3, 2, 1, 0], [1, 1, 1, 1, 1, 1]], np.int32)
    counts, lens = [6, 4, 0, 99, -1], [3, 0, 7, 38, 40]
    want = [t.clone() for t in (k, v, w)]
    new = []
    for s in range(n):
        c = min(max(counts[s], 0), take)
        new.append(min(lens[s] + c, ctx))
        for a in range(c):
            t, row = lens[s] + a, index[s, a]
            if t >= ctx:
                continue
            for x, r in ((want[0], kr), (want[1], vr)):
                x[s, t] = r[s, row].to(x.dtype).to(x.device) if 0 <= row < rows else 0.0
            want[2][s, :, t] = 0.0
    got = jinf_amd.cache_append(k, v, ints(lens), strided(kr, pad), strided(vr, pad), nk,
                                index=ints(index), counts=ints(counts), weights=w)
    assert host(got).tolist() == new
    for a, b in zip((k, v, w), want):
        assert torch.equal(a, b)


def test_append_all_rows_and_none(dev):
    k, v = (rand(i, 3, 20, 128, dtype=torch.float16).cuda() for i in (1, 2))
    kr, vr = (rand(i, 3, 4, 128).cuda() for i in (3, 4))
    wk, wv = k.clone(), v.clone()
    lens = ints([0, 16, 18])
    for s, (t, c) in enumerate(((0, 4), (16, 4), (18, 2))):
        wk[s, t:t + c], wv[s, t:t + c] = kr[s, :c].half(), vr[s, :c].half()
    assert host(jinf_amd.cache_append(k, v, lens, kr, vr, 2)).tolist() == [4, 20, 20]
    assert torch.equal(k, wk) and torch.equal(v, wv)
    none = torch.empty((3, 0, 128), device=dev)
    assert host(jinf_amd.cache_append(k, v, lens, none, none, 2)).tolist() == [0, 16, 18]
    assert torch.equal(k, wk) and torch.equal(v, wv)
    with pytest.raises(JinfError):
        jinf_amd.cache_append(k, v, lens, kr, vr, 2, lens_out=lens)


# ---- evictions ----

def weights_of(kind, n, nk, ctx, seed):
    w = rand(seed, n, nk, ctx).abs()
    if kind == "ties":
        w = torch.round(w * 3.0) / 3.0
    elif kind == "equal":
        w = torch.full_like(w, 0.25)
    elif kind == "odd":  # NaN, infinities, negative numbers, both zeros
        r = np.random.default_rng(seed)
        pick = torch.from_numpy(r.integers(0, 8, size=w.shape))
        for i, x in enumerate((NAN, np.inf, -np.inf, 0.0, -0.0)):
            w[pick == i] = x
        w[pick == 5] *= -1.0
    elif kind == "close":  # neighbours that differ in their last bits
        w = (torch.full_like(w, 1.0).view(torch.int32) +
             torch.from_numpy(np.random.default_rng(seed).integers(0, 700, size=w.shape))
             .to(torch.int32)).view(torch.float32)
    return w


def run_evict(n, ctx, nk, hd, kv, budget, first, recent, lens, kind="plain", place="in", pad=0,
              want_kept=True):
    k, v = (strided(rand(i, n, ctx, nk * hd, dtype=DT[kv]), pad) for i in (1, 2))
    w = strided(weights_of(kind, n, nk, ctx, ctx + budget), pad)
    if place == "in":
        ko, vo, wo, outs = k, v, w, {}
    else:
        rows = min(budget, ctx) + 3
        ko, vo = (strided(rand(i, n, rows, nk * hd, dtype=DT[kv]), pad) for i in (7, 8))
        wo = strided(rand(9, n, nk, rows), pad)
        outs = dict(k_out=ko, v_out=vo, weights_out=wo)
    ki, vi, wi = (host(t).copy() for t in (k, v, w))
    wk, wv, ww = (host(t).copy() for t in (ko, vo, wo))
    want_list = np.full((n, nk, budget), -1, np.int32)
    new = []
    for s in range(n):
        t = min(max(int(lens[s]), 0), ctx)
        m = min(t, budget)
        new.append(m)
        for j in range(nk):
            at = kv_ref.keep(wi[s, j], t, budget, first, recent)
            want_list[s, j, :m] = at
            c = slice(j * hd, (j + 1) * hd)
            wk[s, :m, c], wv[s, :m, c], ww[s, j, :m] = ki[s, at, c], vi[s, at, c], wi[s, j, at]
    kept = torch.full((n, nk, budget), 7, dtype=torch.int32, device="cuda") if want_kept else None
    got = jinf_amd.cache_evict(k, v, w, ints(lens), nk, budget, n_first=first, n_recent=recent,
                               kept=kept, **outs)
    what = f"evict n={n} ctx={ctx} {nk}x{hd} {kv} budget={budget} {kind} {place}"
    say(what)
    assert host(got).tolist() == new, what
    if want_kept:
        assert np.array_equal(host(kept), want_list), what
    for a, b in ((ko, wk), (vo, wv), (wo, ww)):
        assert np.array_equal(host(a), b, equal_nan=True), what
    if place == "out":
        for a, b in ((k, ki), (v, vi), (w, wi)):
            assert np.array_equal(host(a), b, equal_nan=True), "an input changed"


@pytest.mark.parametrize("place", ["in", "out"])
@pytest.mark.parametrize("kv", list(DT))
@pytest.mark.parametrize("n,ctx,nk,hd,budget,first,recent", [
    (1, 1, 1, 64, 1, 0, 0), (1, 5, 1, 64, 1, 0, 0), (2, 100, 2, 64, 99, 4, 10),
    (3, 1200, 8, 128, 512, 4, 128), (1, 5000, 2, 128, 4999, 0, 1), (2, 3000, 1, 64, 7, 3, 4),
    (1, 40000, 1, 64, 5000, 4, 1000), (2, 1024, 3, 64, 1000, 0, 0), (1, 2049, 2, 64, 1025, 1024, 1),
])
def test_evict_shapes(dev, n, ctx, nk, hd, budget, first, recent, kv, place):
    r = np.random.default_rng(ctx + budget)
    lens = [ctx] + [int(x) for x in r.integers(0, ctx + 1, size=n - 1)]
    run_evict(n, ctx, nk, hd, kv, budget, first, recent, lens, place=place)


@pytest.mark.parametrize("place", ["in", "out"])
@pytest.mark.parametrize("kind", ["ties", "equal", "odd", "close"])
def test_evict_weights_of_any_value(dev, kind, place):
    run_evict(2, 3000, 2, 64, "f16", 1500, 4, 100, [3000, 2222], kind=kind, place=place)
    run_evict(2, 900, 2, 64, "f16", 30, 0, 0, [900, 31], kind=kind, place=place, want_kept=False)


@pytest.mark.parametrize("place", ["in", "out"])
def test_evict_lengths(dev, place):
    """Lengths at, below and past the budget and the cache's end, and budgets that
    leave the sums no say."""
    lens = [0, 1, 49, 50, 51, 200, -4, 999]
    run_evict(8, 200, 2, 64, "f16", 50, 2, 20, lens, place=place)
    run_evict(8, 200, 2, 64, "f16", 50, 20, 30, lens, place=place)
    run_evict(8, 200, 2, 64, "f32", 0, 0, 0, lens, place=place)
    run_evict(8, 200, 2, 64, "f32", 500, 5, 5, lens, place=place)


@pytest.mark.parametrize("place", ["in", "out"])
@pytest.mark.parametrize("kv", list(DT))
@pytest.mark.parametrize("hd,pad", [(80, 0), (20, 1), (1, 0), (1000, 0), (128, 8), (64, 3)])
def test_evict_layouts(dev, hd, pad, kv, place):
    run_evict(2, 333, 2, hd, kv, 100, 3, 17, [333, 150], place=place, pad=pad)


@pytest.mark.parametrize("place", ["in", "out"])
def test_evict_long_caches(dev, place):
    """Many chunks move at once, each over rows that others read: the result is the
    copy's."""
    for budget in (9000, 20000, 29990):
        run_evict(2, 30000, 4, 128, "f16", budget, 4, 1000, [30000, 28000], place=place)


def test_evict_into_its_lengths(dev):
    k, v = (rand(i, 2, 50, 128, dtype=torch.float16).cuda() for i in (1, 2))
    w, lens = rand(3, 2, 2, 50).abs().cuda(), ints([50, 4])
    assert jinf_amd.cache_evict(k, v, w, lens, 2, 10, lens_out=lens) is lens
    assert host(lens).tolist() == [10, 4]


def test_evict_into_its_lengths_with_many_workgroups(dev):
    """More (sequence, kv head, plane) triples than run at once: those that start after a
    sequence's new length is stored in place of its old one move its rows all the same."""
    n, ctx, nk, hd, budget = 200, 600, 8, 64, 300
    k, v = (rand(i, n, ctx, nk * hd, dtype=torch.float16).cuda() for i in (1, 2))
    w = rand(3, n, nk, ctx).abs().cuda()
    lens = ints([ctx - 2 * s for s in range(n)])
    ko, vo = (torch.zeros(n, budget, nk * hd, dtype=torch.float16, device="cuda") for _ in range(2))
    wo = torch.zeros(n, nk, budget, device="cuda")
    new = host(jinf_amd.cache_evict(k, v, w, lens, nk, budget, 4, 50, k_out=ko, v_out=vo, weights_out=wo))
    say(f"evict in place into the lengths, {n} sequences")
    jinf_amd.cache_evict(k, v, w, lens, nk, budget, 4, 50, lens_out=lens)
    assert host(lens).tolist() == new.tolist() == [min(ctx - 2 * s, budget) for s in range(n)]
    for s in range(n):
        m = int(new[s])
        assert torch.equal(k[s, :m], ko[s, :m]) and torch.equal(v[s, :m], vo[s, :m]), s
        assert torch.equal(w[s, :, :m], wo[s, :, :m]), s


# ---- together ----

@pytest.mark.parametrize("kv", list(DT))
def test_drafted_decode_over_a_bounded_cache(dev, kv):
    """A bounded cache as a program uses it: decode with summed weights, evict, check
    a drafted tree, append the accepted path, decode again.  The host follows with
    the 64-bit forms on its own copies."""
    n, ctx, nh, nk, hd, T = 3, 96, 8, 2, 64, 9
    dt = DT[kv]
    k, v = (rand(i, n, ctx, nk * hd, dtype=dt).cuda() for i in (1, 2))
    w = torch.zeros(n, nk, ctx, device=dev)
    lens = ints([80, 61, 12])
    hw = np.zeros((n, nk, ctx))
    r = np.random.default_rng(5)
    spent = 0
    for round_ in range(4):
        # decode one token (its own rows appended first)
        kr, vr = rand(40 + round_, n, 1, nk * hd), rand(50 + round_, n, 1, nk * hd)
        lens = jinf_amd.cache_append(k, v, lens, kr.cuda(), vr.cuda(), nk, weights=w)
        q = rand(60 + round_, n, nh * hd, sigma=2.0)
        out = jinf_amd.attention_decode_scored(q.cuda(), k, v, lens, w, nh, nk)
        L = host(lens)
        want, mag, add = kv_ref.scored(q, k.cpu(), v.cpu(), L, nh, nk)
        close(host(out), want, mag, f"round {round_}: decode")
        for s in range(n):
            hw[s, :, L[s] - 1] = 0.0
        hw += add
        spent += 1
        assert np.all(np.abs(host(w) - hw)[:, :, :][add > 0] <=
                      (2e-5 * hw + spent * 2.0 ** -24 * hw + 1e-30)[add > 0])
        # the positions that stay are those of the device's own sums
        hwd = host(w)
        kept = torch.empty((n, nk, 40), dtype=torch.int32, device=dev)
        lens = jinf_amd.cache_evict(k, v, w, lens, nk, 40, n_first=2, n_recent=10, kept=kept)
        at = host(kept)
        for s in range(n):
            m = min(int(L[s]), 40)
            for j in range(nk):
                assert np.array_equal(at[s, j, :m], kv_ref.keep(hwd[s, j], int(L[s]), 40, 2, 10))
                hw[s, j, :m] = hw[s, j, at[s, j, :m]]
        # a drafted tree, and the path from its last node
        par = np.stack([r.integers(-1, i, size=n) if i else np.full(n, -1) for i in range(T)], 1)
        mask = jinf_amd.tree_mask(par)
        qd, kd, vd = (rand(70 + 10 * round_ + i, n, T, x * hd) for i, x in enumerate((nh, nk, nk)))
        got = jinf_amd.attention_tree(qd.cuda(), k, v, lens, kd.cuda(), vd.cuda(), mask, nh, nk)
        want, mag = kv_ref.tree(qd, k.cpu(), v.cpu(), host(lens), kd, vd, mask, nh, nk)
        close(host(got), want, mag, f"round {round_}: tree")
        bits = kv_ref.mask_bits(mask)[:, T - 1]
        path = [np.flatnonzero(b) for b in bits]
        depth = max(map(len, path))
        index = np.zeros((n, depth), np.int32)
        for s in range(n):
            index[s, :len(path[s])] = path[s]
        before = host(lens)
        lens = jinf_amd.cache_append(k, v, lens, kd.cuda(), vd.cuda(), nk, index=ints(index),
                                     counts=ints([len(p) for p in path]), weights=w)
        for s in range(n):
            m = len(path[s])
            hw[s, :, before[s]:before[s] + m] = 0.0
            assert torch.equal(k[s, before[s]:before[s] + m].cpu(), kd[s, path[s]].to(dt))
        # the accepted path's last node, decoded as a plain token, agrees with its tree row
        a = host(jinf_amd.attention_decode(qd[:, T - 1].contiguous().cuda(), k, v, lens, nh, nk))
        assert np.all(np.abs(a - host(got)[:, T - 1].astype(np.float64)) <= 4e-5 * mag[:, T - 1])


@pytest.mark.parametrize("kv", list(DT))
def test_replayed_graph_and_other_stream(dev, kv):
    """One step of all four operators captured in a graph and replayed with eager work
    between, and run on another stream: the eager bits each time."""
    n, ctx, nh, nk, hd, T = 2, 1400, 8, 2, 128, 5
    dt = DT[kv]
    k0, v0 = (rand(i, n, ctx, nk * hd, dtype=dt).cuda() for i in (1, 2))
    w0 = rand(3, n, nk, ctx).abs().cuda()
    q, kd, vd = (rand(4 + i, n, T, x * hd).cuda() for i, x in enumerate((nh, nk, nk)))
    mask = random_mask(np.random.default_rng(1), n, T)
    k, v, w = k0.clone(), v0.clone(), w0.clone()
    l0 = ints([1300, 900])
    l1, l2 = torch.empty_like(l0), torch.empty_like(l0)
    out, o1 = torch.empty_like(q), torch.empty(n, nh * hd, device=dev)
    tws = jinf_amd.attention_tree_workspace(n, T, nh, nk, hd, ctx)
    sws = jinf_amd.attention_scored_workspace(n, nh, nk, hd, ctx)
    ews = jinf_amd.cache_evict_workspace(n, nk, 800)
    kept = torch.empty((n, nk, 800), dtype=torch.int32, device=dev)
    q1 = q[:, 0].contiguous()

    def step():
        jinf_amd.attention_tree(q, k, v, l0, kd, vd, mask, nh, nk, out=out, workspace=tws)
        jinf_amd.cache_append(k, v, l0, kd, vd, nk, weights=w, lens_out=l1)
        jinf_amd.attention_decode_scored(q1, k, v, l1, w, nh, nk, out=o1, workspace=sws)
        jinf_amd.cache_evict(k, v, w, l1, nk, 800, n_first=4, n_recent=100, lens_out=l2, kept=kept,
                             workspace=ews)

    def reset():
        for a, b in ((k, k0), (v, v0), (w, w0)):
            a.copy_(b)
        for t in (out, o1):
            t.fill_(NAN)
        for t in (l1, l2, kept):
            t.fill_(-9)

    def state():
        return [host(t).copy() for t in (k, v, w, out, o1, l1, l2, kept)]

    reset()
    step()
    want = state()
    reset()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for i in range(4):
        reset()
        for t in (tws, sws, ews):
            t.fill_(255 * (i % 2))  # a workspace's old contents do not matter
        _ = (w0 * 2).sum()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(state(), want):
            assert np.array_equal(a, b), f"replay {i}"
    reset()
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        step()
    stream.synchronize()
    for a, b in zip(state(), want):
        assert np.array_equal(a, b), "another stream"


def test_repeatable_bits(dev):
    """Two runs on the same inputs give the same bits."""
    n, ctx, nh, nk, hd, T = 4, 6000, 32, 8, 128, 30
    k, v = (rand(i, n, ctx, nk * hd, dtype=torch.float16).cuda() for i in (1, 2))
    q, kd, vd = (rand(4 + i, n, T, x * hd).cuda() for i, x in enumerate((nh, nk, nk)))
    lens, mask = ints([6000, 5000, 20, 0]), random_mask(np.random.default_rng(1), n, T)
    a = host(jinf_amd.attention_tree(q, k, v, lens, kd, vd, mask, nh, nk)).copy()
    b = host(jinf_amd.attention_tree(q, k, v, lens, kd, vd, mask, nh, nk))
    assert np.array_equal(a, b)
