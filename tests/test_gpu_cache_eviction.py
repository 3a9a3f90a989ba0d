"""Eviction: the choice of the tokens that stay (whole numbers: equal to a plain sort) and the move of their rows (bytes: equal to a plain gather;
a scaled E4M3 block equal, bit for bit, to the rule written out in NumPy's IEEE single precision)."""
import ctypes

import numpy as np
import pytest

from tempura_b200 import _native as N

pytestmark = pytest.mark.gpu
BS = 16


@pytest.fixture(scope="module")
def H():
    import torch
    assert torch.cuda.is_available()
    from tempura_b200 import handoff
    return handoff


def plain_choice(row, length, protect, budget, recent):
    protect = min(protect, length)
    n = length if protect + recent >= length or budget >= length else max(budget, protect + recent)
    if n == length:
        return list(range(length))
    mid = np.arange(protect, length - recent)
    key = row[mid].astype(np.float64)
    key = np.where(np.isnan(key), -np.inf, key)
    rank = np.lexsort((mid, np.isnan(row[mid]), -key))              # score down, numbers before NaN, then index
    return sorted(list(range(protect)) + [int(i) for i in mid[rank[: n - protect - recent]]] + list(range(length - recent, length)))


def check_choice(H, scores, lens, protect, budget, recent, kept_width=None):
    import torch
    s = torch.from_numpy(scores).cuda()
    width = kept_width or max(1, max(len(plain_choice(scores[0, i, 0], lens[i], protect[i], budget, recent)) for i in range(len(lens))))
    kept = torch.full(scores.shape[:3] + (width,), -7, dtype=torch.int32).cuda()
    ev = H.CacheEviction(None, None, torch.tensor(lens, dtype=torch.int32).cuda(), s, budget, recent,
                         protect=torch.tensor(protect, dtype=torch.int32).cuda(), kept=kept)
    got, new = ev.select()
    got, new = got.cpu().numpy(), new.cpu().numpy()
    assert int(ev.status.item()) == 0
    for layer in range(scores.shape[0]):
        for i, length in enumerate(lens):
            for h in range(scores.shape[2]):
                want = plain_choice(scores[layer, i, h], length, protect[i], budget, recent)
                assert new[i] == len(want)
                assert got[layer, i, h, : len(want)].tolist() == want, (layer, i, h)
                assert (got[layer, i, h, len(want):] == -7).all()      # behind the end: left alone
    return new


@pytest.mark.parametrize("budget,recent", [(1, 0), (7, 7), (20, 5), (64, 64), (200, 16), (5000, 3), (100, 0), (3, 40)])
def test_select_matches_a_plain_sort(H, budget, recent):
    rng = np.random.default_rng(budget)
    lens = [0, 1, 2, 31, 32, 33, 100, 512, 513, 1500]
    scores = (rng.exponential(size=(2, len(lens), 3, 1501)) ** 3).astype(np.float32)
    scores[:, :, 1] = np.round(scores[:, :, 1], 1)                    # many ties
    scores[:, :, 2] = 0.25                                            # all tied: the first ones stay
    check_choice(H, scores, lens, [0, 1, 0, 16, 0, 40, 5, 0, 32, 48], budget, recent)


def test_select_orders_zeros_infinities_nans_and_denormals(H):
    rng = np.random.default_rng(3)
    pool = np.array([0.0, -0.0, np.inf, -np.inf, np.nan, -np.nan, 1e-45, -1e-45, 1.0, -1.0, 3e38, -3e38, 1.0000001], dtype=np.float32)
    scores = pool[rng.integers(0, len(pool), size=(1, 4, 2, 700))]
    for budget in (1, 50, 150, 300, 690):
        check_choice(H, scores, [700, 699, 350, 691], [0, 3, 0, 16], budget, 10 if budget > 10 else 0)


@pytest.mark.parametrize("shape,lens", [((1, 1, 1, 70001), [70001]), ((1, 2, 2, 30000), [30000, 17]), ((3, 1, 4, 9000), [8999]), ((1, 1, 1, 400003), [400003])])
def test_select_splits_long_rows_over_a_cluster(H, shape, lens):
    """Few long rows: a cluster per row, the longest too long for its CTAs' shared memory; ties across CTAs go to the lower index."""
    rng = np.random.default_rng(9)
    scores = rng.random(shape, dtype=np.float32)
    scores[scores < 0.5] = 0.0
    scores[:, :, 0] = np.round(scores[:, :, 0], 2)
    for budget in (100, shape[3] // 3, shape[3] - 5):
        check_choice(H, scores, lens, [0] * len(lens), budget, 64)


def test_select_does_not_cut_what_kept_cannot_hold(H):
    import torch
    scores = torch.rand((1, 2, 1, 300)).cuda()
    ev = H.CacheEviction(None, None, torch.tensor([300, 300], dtype=torch.int32).cuda(), scores, 40, 10,
                         protect=torch.tensor([100, 0], dtype=torch.int32).cuda())
    kept, new = ev.select()
    assert new.tolist() == [300, 40]
    assert int(ev.status.item()) == N.ERR_INVALID_CONFIG


# ---- compact ------------------------------------------------------------------------------------------------------------------------
def enc(x):
    """f32 -> E4M3 bytes: to nearest even, below 2^-6 to a signed zero (|x| <= 448 here)."""
    import torch
    t = torch.from_numpy(np.ascontiguousarray(x))
    t = torch.where(t.abs() < 2.0 ** -6, t * 0.0, t)
    return t.to(torch.float8_e4m3fn).view(torch.uint8).numpy()


def dec(b):
    import torch
    return torch.from_numpy(np.ascontiguousarray(b)).view(torch.float8_e4m3fn).float().numpy()


def make(H, dtype, layers, lens, heads, dim, seed, shared_blocks=0):
    """A pool whose every byte is set, tables over shuffled blocks; the first `shared_blocks` blocks are the same for all sequences."""
    import torch
    rng = np.random.default_rng(seed)
    width = max(1, max((t + BS - 1) // BS for t in lens))
    need = shared_blocks + sum(max(0, (t + BS - 1) // BS - shared_blocks) for t in lens) + 3
    ids = rng.permutation(need).tolist()
    common = [ids.pop() for _ in range(shared_blocks)]
    tables = np.full((len(lens), width), -1, dtype=np.int64)
    for s, t in enumerate(lens):
        nb = (t + BS - 1) // BS
        row = common[:nb] + [ids.pop() for _ in range(nb - min(nb, shared_blocks))]
        tables[s, :nb] = row
    pool = H.Pool.allocate(0, layers, heads, dim, BS, need, "f16" if dtype == "f16" else "e4m3", scales=dtype == "e4m3")
    for layer in range(layers):
        for is_v in (False, True):
            if dtype == "f16":
                raw = rng.integers(0, 65536, size=(need, BS, heads, dim)).astype(np.uint16)       # any bits, NaN payloads among them
                pool.blocks(layer, is_v).copy_(torch.from_numpy(raw.view(np.float16)))
                pool.blocks(layer, is_v).view(torch.int16).copy_(torch.from_numpy(raw.view(np.int16)))
            else:
                raw = enc((rng.standard_normal((need, BS, heads, dim)) * 100).clip(-448, 448).astype(np.float32))
                pool.blocks(layer, is_v).copy_(torch.from_numpy(raw))
            if dtype == "e4m3":
                sc = (rng.random((need, heads)) * 0.01 + 1e-4).astype(np.float32)
                sc[::4] = np.float32(0.005)                           # equal scales: those rows keep their bytes
                (pool.v_scales if is_v else pool.k_scales)[layer].copy_(torch.from_numpy(sc))
    return pool, tables


def snapshot(pool):
    out = {}
    for layer in range(pool.n_layers):
        for is_v in (False, True):
            x = pool.blocks(layer, is_v)
            out[layer, is_v] = x.cpu().numpy().view(np.uint16 if x.element_size() == 2 else np.uint8).copy()
            if pool.k_scales is not None:
                out[layer, is_v, "s"] = (pool.v_scales if is_v else pool.k_scales)[layer].cpu().numpy().copy()
    return out


def plain_compact(before, layers, heads, tables, lens, kept, new, scaled):
    after = {k: v.copy() for k, v in before.items()}
    for layer in range(layers):
        for is_v in (False, True):
            old, x = before[layer, is_v], after[layer, is_v]
            for s, length in enumerate(lens):
                if new[s] == length:
                    continue
                for h in range(heads):
                    for b in range((new[s] + BS - 1) // BS):
                        js = range(b * BS, min(new[s], b * BS + BS))
                        src = [int(kept[layer, s, h, j]) for j in js]
                        if all(k == j for k, j in zip(src, js)):
                            continue
                        dst = tables[s, b]
                        rows = [old[tables[s, k // BS], k % BS, h] for k in src]
                        if scaled:
                            sc = [before[layer, is_v, "s"][tables[s, k // BS], h] for k in src]
                            top = max(sc)
                            rows = [r if c == top else enc(dec(r) * np.float32(c / top)) for r, c in zip(rows, sc)]
                            after[layer, is_v, "s"][dst, h] = top
                        for j, r in zip(js, rows):
                            x[dst, j % BS, h] = r
    return after


@pytest.mark.parametrize("dtype", ["f16", "e4m3", "e4m3 unscaled"])
@pytest.mark.parametrize("heads,dim", [(4, 128), (3, 64), (1, 128)])
@pytest.mark.parametrize("budget,recent,shared", [(40, 8, 0), (100, 0, 2), (1, 0, 0), (333, 50, 3)])
def test_compact_moves_the_kept_rows(H, dtype, heads, dim, budget, recent, shared):
    import torch
    layers, lens = 2, [0, 5, 48, 300, 777, 1100]
    pool, tables = make(H, dtype, layers, lens, heads, dim, seed=budget + heads, shared_blocks=shared)
    rng = np.random.default_rng(1)
    start = (rng.random((layers, len(lens), heads, 1200)) ** 4).astype(np.float32)
    scores = torch.from_numpy(start.copy()).cuda()
    dev_lens = torch.tensor(lens, dtype=torch.int32).cuda()
    protect = torch.full((len(lens),), shared * BS, dtype=torch.int32).cuda()
    ev = H.CacheEviction(pool, torch.from_numpy(tables.astype(np.int32)).cuda(), dev_lens, scores, budget, recent, protect=protect)
    before = snapshot(pool)
    ev.evict()
    assert int(ev.status.item()) == 0
    kept, new = ev.kept.cpu().numpy(), ev.new_lens.cpu().numpy()
    assert dev_lens.tolist() == new.tolist()
    want = plain_compact(before, layers, heads, tables, lens, kept, new, dtype == "e4m3")
    got = snapshot(pool)
    for k in want:
        assert np.array_equal(got[k], want[k]), k                     # every byte of the pool, the untouched blocks among them
    sc = scores.cpu().numpy()
    for layer in range(layers):
        for s, length in enumerate(lens):
            for h in range(heads):
                w = start[layer, s, h].copy()
                if new[s] < length:
                    w[: new[s]] = start[layer, s, h, kept[layer, s, h, : new[s]]]
                    w[new[s]: length] = 0
                assert np.array_equal(sc[layer, s, h], w)
    # a second cut of what is left
    ev2 = H.CacheEviction(pool, torch.from_numpy(tables.astype(np.int32)).cuda(), dev_lens, scores, max(1, budget // 2), recent // 2, protect=protect)
    lens2, before = dev_lens.tolist(), snapshot(pool)
    ev2.evict()
    want = plain_compact(before, layers, heads, tables, lens2, ev2.kept.cpu().numpy(), ev2.new_lens.cpu().numpy(), dtype == "e4m3")
    got = snapshot(pool)
    for k in want:
        assert np.array_equal(got[k], want[k]), k


def test_compact_long_sequence_walks_many_tiles(H):
    import torch
    lens = [9000]
    pool, tables = make(H, "f16", 1, lens, 2, 128, seed=5)
    scores = torch.rand((1, 1, 2, 9000), generator=torch.Generator().manual_seed(2)).cuda()
    ev = H.CacheEviction(pool, torch.from_numpy(tables.astype(np.int32)).cuda(), torch.tensor(lens, dtype=torch.int32).cuda(), scores, 8000, 100)
    before = snapshot(pool)
    ev.evict()
    want = plain_compact(before, 1, 2, tables, lens, ev.kept.cpu().numpy(), ev.new_lens.cpu().numpy(), False)
    got = snapshot(pool)
    assert all(np.array_equal(got[k], want[k]) for k in want)


def test_compact_reports_and_skips_what_it_cannot_trust(H):
    import torch
    lens = [100]
    pool, tables = make(H, "f16", 1, lens, 1, 64, seed=6)
    dev = torch.from_numpy(tables.astype(np.int32)).cuda()
    ev = H.CacheEviction(pool, dev, torch.tensor(lens, dtype=torch.int32).cuda(), torch.rand((1, 1, 1, 100)).cuda(), 20, 0)
    ev.select()
    kept = ev.kept.clone()
    kept[0, 0, 0, 5], kept[0, 0, 0, 6], kept[0, 0, 0, 7] = 1 << 30, 3, 100   # outside, below its place, one past the end
    ev.kept.copy_(kept)
    before = snapshot(pool)
    ev.compact()
    assert int(ev.status.item()) == N.ERR_INVALID_CONFIG
    k = kept.cpu().numpy().copy()
    k[0, 0, 0, 5:8] = [5, 6, 7]                                       # those rows stay
    want = plain_compact(before, 1, 1, tables, lens, k, [20], False)
    got = snapshot(pool)
    assert all(np.array_equal(got[x], want[x]) for x in want)
    ev.status.zero_()
    bad = dev.clone()
    bad[0, 0] = 1 << 24                                               # the first destination block is foreign: nothing is written there
    before = snapshot(pool)
    ev2 = H.CacheEviction(pool, bad, torch.tensor(lens, dtype=torch.int32).cuda(), torch.rand((1, 1, 1, 100)).cuda(), 10, 0)
    ev2.select()
    ev2.compact()
    assert int(ev2.status.item()) == N.ERR_INVALID_CONFIG
    got = snapshot(pool)
    assert all(np.array_equal(got[x], before[x]) for x in before)


def test_eviction_in_a_graph(H):
    import torch
    lens = [200, 64]
    pool, tables = make(H, "f16", 2, lens, 2, 64, seed=7)
    dev_lens = torch.tensor(lens, dtype=torch.int32).cuda()
    scores = torch.rand((2, 2, 2, 256), generator=torch.Generator().manual_seed(4)).cuda()
    ev = H.CacheEviction(pool, torch.from_numpy(tables.astype(np.int32)).cuda(), dev_lens, scores, 50, 5)
    before, start = snapshot(pool), scores.clone()
    graph = torch.cuda.CUDAGraph()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        with torch.cuda.graph(graph, stream=side):
            ev.evict()
    torch.cuda.synchronize()
    assert dev_lens.tolist() == lens                                   # captured, not run
    graph.replay()
    torch.cuda.synchronize()
    assert dev_lens.tolist() == [50, 50]
    want = plain_compact(before, 2, 2, tables, lens, ev.kept.cpu().numpy(), [50, 50], False)
    got = snapshot(pool)
    assert all(np.array_equal(got[x], want[x]) for x in want)
    graph.replay()                                                      # nothing left to cut
    assert dev_lens.tolist() == [50, 50]
    again = snapshot(pool)
    assert all(np.array_equal(got[x], again[x]) for x in got)
    assert not torch.equal(start, scores)


def test_eviction_refusals(H):
    import torch
    pool, tables = make(H, "f16", 1, [40], 2, 64, seed=8)
    ev = H.CacheEviction(pool, torch.from_numpy(tables.astype(np.int32)).cuda(), torch.tensor([40], dtype=torch.int32).cuda(),
                         torch.rand((1, 1, 2, 40)).cuda(), 10, 2)

    def call(fn, args, change, pool_c=None):
        a = type(args).from_buffer_copy(args)
        for k, v in change.items():
            setattr(a, k, v)
        rc = fn(ctypes.byref(pool_c), ctypes.byref(a), None) if pool_c is not None else fn(ctypes.byref(a), None)
        return rc
    sel, cmp_ = N.lib().tkv_evict_select_enqueue, N.lib().tkv_evict_compact_enqueue
    assert call(sel, ev._select, {}) == 0 and call(sel, ev._select, {"n_seqs": 0}) == 0
    for change in ({"scores": 0}, {"kv_lens": 0}, {"kept": 0}, {"new_lens": 0}, {"scores": ev._select.scores + 2}):
        assert call(sel, ev._select, change) == N.ERR_INVALID_CONFIG, change
    for change in ({"score_stride": 39}, {"kept_stride": 9}, {"budget": 11}):
        assert call(sel, ev._select, change) == N.ERR_DIMENSION_MISMATCH, change
    assert call(cmp_, ev._compact, {"n_layers": 0}, ev._pool_c) == 0
    for change in ({"layer_begin": 1}, {"tables": 0}, {"kept": 0}, {"kv_lens": 0}, {"new_lens": 0}):
        assert call(cmp_, ev._compact, change, ev._pool_c) == N.ERR_INVALID_CONFIG, change
    for change in ({"table_stride": 2}, {"score_stride": 39}):
        assert call(cmp_, ev._compact, change, ev._pool_c) == N.ERR_DIMENSION_MISMATCH, change
    with pytest.raises(N.TkvError):
        H.CacheEviction(None, None, ev.kv_lens, ev.scores, 10, 2).compact()
