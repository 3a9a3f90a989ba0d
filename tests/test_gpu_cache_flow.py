"""The cache operators together, as a decode loop under memory pressure uses them: prompts resolved against the device prefix index,
pages from the device allocator, steps of scored attention, eviction, pages given back, shared-prefix attention over what is left."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu
BS = 16


def test_decode_loop_scores_evicts_frees_and_goes_on():
    import torch
    from tempura_b200 import handoff as H
    layers, heads, dim, group, total = 2, 4, 64, 8, 256
    prefix, budget, recent = 64, 128, 16
    lens = [200, 90, 333, 64, 129]                                      # the fourth is the prefix alone
    n, width = len(lens), 24
    g = torch.Generator().manual_seed(1)
    pool = H.Pool.allocate(0, layers, heads, dim, BS, total, "f16", refcounts=True)
    index, alloc = H.PrefixIndex(0, 1024, BS), H.DevicePageAllocator(0, total)
    shared = torch.randint(0, 30000, (prefix,), generator=g, dtype=torch.int32)
    tokens = torch.randint(0, 30000, (n, width * BS), generator=g, dtype=torch.int32)
    tokens[:, :prefix] = shared
    tokens, dev_lens = tokens.cuda(), torch.tensor(lens, dtype=torch.int32).cuda()
    tables = torch.full((n, width), -1, dtype=torch.int32).cuda()
    # the prefix is already cached: its pages are in the index
    seed_table = torch.full((1, width), -1, dtype=torch.int32).cuda()
    alloc.allocate(seed_table, counts=torch.tensor([prefix // BS], dtype=torch.int32).cuda())
    index.insert(tokens[:1, :prefix].contiguous(), torch.tensor([prefix], dtype=torch.int32).cuda(), seed_table[:, : prefix // BS].contiguous())
    matched, _ = index.lookup(tokens, dev_lens, out_pages=tables)
    assert matched.tolist() == [prefix // BS] * n
    alloc.allocate(tables, first=matched, seq_lens=dev_lens, block_size=BS)
    assert int(alloc.status.item()) == 0
    free_before = alloc.available()
    # prefill: every position's K and V, the prefix once
    host = tables.cpu().numpy()
    values = {}
    for layer in range(layers):
        for is_v in (False, True):
            x = (torch.randn((total, BS, heads, dim), generator=g) * 0.7).to(torch.float16)
            pool.blocks(layer, is_v).copy_(x)
            values[layer, is_v] = x.double()
    cache = {}                                                           # (layer, is_v, sequence, head) -> rows in order
    for s, t in enumerate(lens):
        at = [(host[s, i // BS], i % BS) for i in range(t)]
        for layer in range(layers):
            for is_v in (False, True):
                for h in range(heads):
                    cache[layer, is_v, s, h] = torch.stack([values[layer, is_v][b, o, h] for b, o in at])
    # decode steps that accumulate weights
    scores = torch.zeros((layers, n, heads, width * BS)).cuda()
    want_scores = {(layer, s, h): torch.zeros(lens[s], dtype=torch.float64) for layer in range(layers) for s in range(n) for h in range(heads)}
    scale = 1 / np.sqrt(dim)

    def attend(layer, s, q, w_out=None):
        out = torch.zeros((heads * group, dim), dtype=torch.float64)
        for h in range(heads):
            k, v = cache[layer, False, s, h], cache[layer, True, s, h]
            w = torch.softmax(q[h * group:(h + 1) * group].double() @ k.T * scale, dim=1)
            out[h * group:(h + 1) * group] = w @ v
            if w_out is not None:
                w_out[layer, s, h] += w.sum(dim=0)
        return out
    dq = torch.empty((n, heads * group, dim), dtype=torch.float16).cuda()
    scored = H.ScoredDecodeAttention(pool, dq, tables, dev_lens, scores, width * BS)
    for step in range(3):
        q = (torch.randn((n, heads * group, dim), generator=g) * 2).to(torch.float16)
        dq.copy_(q)
        for layer in range(layers):
            out = scored.enqueue(layer).double().cpu()
            for s in range(n):
                assert (out[s] - attend(layer, s, q[s], want_scores)).abs().max() < 3e-3
    assert int(scored.status.item()) == 0
    for (layer, s, h), w in want_scores.items():
        assert torch.allclose(scores[layer, s, h, : lens[s]].double().cpu(), w, rtol=1e-4, atol=1e-6)
    # eviction: the shared prefix is protected
    protect = torch.full((n,), prefix, dtype=torch.int32).cuda()
    before = pool.blocks(0).clone()
    old_lens = dev_lens.clone()
    ev = H.CacheEviction(pool, tables, dev_lens, scores, budget, recent, protect=protect)
    new = ev.evict().tolist()
    assert int(ev.status.item()) == 0 and new == [128, 90, 128, 64, 128] and dev_lens.tolist() == new
    assert torch.equal(pool.blocks(0)[host[0, : prefix // BS]], before[host[0, : prefix // BS]])
    kept = ev.kept.cpu().numpy()
    for (layer, s, h), w in want_scores.items():
        if new[s] < lens[s]:
            idx = kept[layer, s, h, : new[s]].tolist()
            assert idx[:prefix] == list(range(prefix)) and idx[-recent:] == list(range(lens[s] - recent, lens[s])) and idx == sorted(set(idx))
            out = [i for i in range(prefix, lens[s] - recent) if i not in set(idx)]
            assert max(float(w[i]) for i in out) <= min(float(w[i]) for i in idx[prefix:-recent]) * (1 + 1e-4) + 1e-6
            for is_v in (False, True):
                cache[layer, is_v, s, h] = cache[layer, is_v, s, h][idx]
    # the blocks behind the new lengths go back
    first = (dev_lens + BS - 1) // BS
    alloc.free(tables, first=first.to(torch.int32), seq_lens=old_lens, block_size=BS)
    assert int(alloc.status.item()) == 0
    gone = sum((a + BS - 1) // BS - (b + BS - 1) // BS for a, b in zip(lens, new))
    assert gone > 0 and alloc.available() == free_before + gone
    # the batch goes on: prefix attention over what is left, and a scored step that agrees with it
    q = (torch.randn((n, heads * group, dim), generator=g) * 2).to(torch.float16)
    dq.copy_(q)
    pre = H.PrefixAttention(pool, dq, tables, dev_lens, torch.tensor([0, n], dtype=torch.int32).cuda(), torch.tensor([prefix], dtype=torch.int32).cuda(),
                            width * BS, prefix)
    for layer in range(layers):
        out, again = pre.enqueue(layer).double().cpu(), scored.enqueue(layer).double().cpu()
        for s in range(n):
            want = attend(layer, s, q[s])
            assert (out[s] - want).abs().max() < 4e-3 and (again[s] - want).abs().max() < 3e-3
    assert int(pre.status.item()) == 0
    index.close()
    alloc.close()
