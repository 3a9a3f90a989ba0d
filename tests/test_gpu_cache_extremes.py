"""The cache operators at the ends of their ranges: head counts that no benchmark has, more groups and sequences than a CTA has threads, empty groups and
batches, more layers than a launch takes, blocks whose byte offsets pass 32 bits, negative scales."""
import pytest

from test_gpu_cache_eviction import make, plain_compact, snapshot
from test_gpu_cache_operators import BS, H, Cache, out_close, prefix_case, scores_close  # noqa: F401  (H is the fixture)

pytestmark = pytest.mark.gpu


def i32(v):
    import torch
    return torch.tensor(v, dtype=torch.int32).cuda()


@pytest.mark.parametrize("dtype", ["f16", "e4m3"])
@pytest.mark.parametrize("kv_heads,head_dim,group", [(9, 64, 1), (17, 128, 2), (64, 64, 2), (130, 64, 1)])
def test_attention_over_many_kv_heads(H, dtype, kv_heads, head_dim, group):  # noqa: F811
    import torch
    lens = [1, 40, 0, 16, 133]
    c = Cache(H, lens, kv_heads, head_dim, dtype, seed=kv_heads)
    q = torch.randn((len(lens), kv_heads * group, head_dim), generator=torch.Generator().manual_seed(1)).to(torch.float16)
    scores = torch.zeros((1, len(lens), kv_heads, 136)).cuda()
    attn = H.ScoredDecodeAttention(c.pool, q.cuda(), c.dev_tables, c.dev_lens, scores, 136)
    out = attn.enqueue(0)
    assert int(attn.status.item()) == 0
    for s, (want, w, vmax) in enumerate(c.attention(0, q, attn.sm_scale)):
        out_close(out[s], want, vmax, False)
        if lens[s]:
            w = w.view(kv_heads, group, lens[s]).sum(dim=1)
            scores_close(scores[0, s, :, : lens[s]], w, torch.zeros_like(w))
    c, q, attn, lens = prefix_case(H, dtype, kv_heads, head_dim, group, [3, 2], [144, 32], [0, 5, 20], seed=kv_heads + 1)
    out = attn.enqueue(0)
    assert int(attn.status.item()) == 0
    for s, (want, _, vmax) in enumerate(c.attention(0, q, attn.sm_scale)):
        out_close(out[s], want, vmax, False)


@pytest.mark.parametrize("dtype", ["f16", "e4m3"])
def test_prefix_attention_with_more_groups_and_sequences_than_a_cta_has_threads(H, dtype):  # noqa: F811
    """1 300 groups of 0 to 3 members (many empty), some 2 000 sequences, most with a prefix of one or two blocks."""
    sizes = [(g * 7919) % 4 for g in range(1300)]
    prefixes = [16 * (g % 3) for g in range(1300)]
    c, q, attn, lens = prefix_case(H, dtype, 2, 64, 2, sizes, prefixes, [0, 3, 17, 1], seed=3)
    out = attn.enqueue(0)
    assert int(attn.status.item()) == 0
    for s, (want, _, vmax) in enumerate(c.attention(0, q, attn.sm_scale)):
        out_close(out[s], want, vmax, False)


def test_prefix_attention_empty_groups_and_an_empty_batch(H):  # noqa: F811
    import torch
    c, q, attn, lens = prefix_case(H, "f16", 2, 128, 4, [0, 3, 0, 0, 2, 0], [64, 48, 16, 0, 0, 64], [2, 30], seed=4)
    out = attn.enqueue(0)
    assert int(attn.status.item()) == 0
    for s, (want, _, vmax) in enumerate(c.attention(0, q, attn.sm_scale)):
        out_close(out[s], want, vmax, False)
    attn.kv_lens.zero_()
    attn.out.fill_(3.0)
    assert (attn.enqueue(0) == 0).all() and int(attn.status.item()) == 0
    attn.group_starts.zero_()                                          # no sequence in any group
    attn.out.fill_(3.0)
    assert (attn.enqueue(0) == 3.0).all() and int(attn.status.item()) == 0
    scores = torch.full((1, 5, 2, 80), 0.5).cuda()
    scored = H.ScoredDecodeAttention(c.pool, attn.q, c.dev_tables, attn.kv_lens, scores, 0)
    assert (scored.enqueue(0) == 0).all() and int(scored.status.item()) == 0 and (scores == 0.5).all()


@pytest.mark.parametrize("dtype", ["f16", "e4m3", "e4m3 unscaled"])
def test_attention_with_a_negative_scale(H, dtype):  # noqa: F811
    import torch
    c, q, attn, lens = prefix_case(H, dtype, 3, 128, 4, [5, 40], [160, 400], [5, 0, 70], seed=9)
    neg = H.PrefixAttention(c.pool, attn.q, attn.tables, attn.kv_lens, attn.group_starts, attn.prefix_lens, max(lens), 400, sm_scale=-0.11)
    scored = H.ScoredDecodeAttention(c.pool, attn.q, c.dev_tables, attn.kv_lens, torch.zeros((1, len(lens), 3, max(lens))).cuda(), max(lens), sm_scale=-0.11)
    for a in (neg, scored):
        out = a.enqueue(0)
        assert int(a.status.item()) == 0
        for s, (want, _, vmax) in enumerate(c.attention(0, q, -0.11)):
            out_close(out[s], want, vmax, False)


@pytest.mark.parametrize("dtype", ["f16", "e4m3"])
def test_blocks_whose_offsets_pass_32_bits(H, dtype):  # noqa: F811
    """K and V of 4.8 GB each: the sequences' blocks lie at both ends."""
    import torch
    kv_heads, dim, es = 8, 128, 2 if dtype == "f16" else 1
    total = 4_800_000_000 // (BS * kv_heads * dim * es)
    lens = [300, 77, 64]
    small = Cache(H, lens, kv_heads, dim, dtype, seed=12)
    n = small.pool.total_blocks
    pool = H.Pool.allocate(0, 1, kv_heads, dim, BS, total, "f16" if dtype == "f16" else "e4m3", scales=dtype == "e4m3", fill_byte=None)
    place = torch.tensor([b if b % 3 == 0 else total - 1 - b for b in range(n)]).cuda()
    for is_v in (False, True):
        pool.blocks(0, is_v)[place] = small.pool.blocks(0, is_v)
        if dtype == "e4m3":
            (pool.v_scales if is_v else pool.k_scales)[0, place] = (small.pool.v_scales if is_v else small.pool.k_scales)[0]
    live = small.dev_tables >= 0
    tables = torch.where(live, place[small.dev_tables.clamp_min(0).long()].to(torch.int32), small.dev_tables)
    q = torch.randn((3, 32, dim), generator=torch.Generator().manual_seed(2)).to(torch.float16)
    scores = torch.rand((1, 3, kv_heads, 304), generator=torch.Generator().manual_seed(3)).cuda()
    handles = []
    for p, t in ((small.pool, small.dev_tables), (pool, tables)):
        sc = scores.clone()
        lens_d = small.dev_lens.clone()
        scored = H.ScoredDecodeAttention(p, q.cuda(), t, lens_d, sc, 300)
        pre = H.PrefixAttention(p, q.cuda(), t, lens_d, i32([0, 1, 2, 3]), i32([256, 0, 64]), 300, 256)
        outs = [scored.enqueue(0).clone(), pre.enqueue(0).clone()]
        ev = H.CacheEviction(p, t, lens_d, sc, 100, 10)
        new = ev.evict().tolist()
        assert [int(h.status.item()) for h in (scored, pre, ev)] == [0, 0, 0] and new == [100, 77, 64]
        after = [p.blocks(0, is_v)[t[s, : (new[s] + BS - 1) // BS].long()].view(torch.uint8).clone() for is_v in (False, True) for s in range(3)]
        handles.append((outs, sc, after))
    (outs, sc, after), (outs2, sc2, after2) = handles
    for s, (want, _, vmax) in enumerate(small.attention(0, q, 1 / dim ** 0.5)):
        out_close(outs[0][s], want, vmax, False)
    for a, b in zip(outs + [sc] + after, outs2 + [sc2] + after2):      # where the blocks lie changes no bit
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", ["f16", "e4m3"])
def test_eviction_of_more_layers_than_a_launch_takes(H, dtype):  # noqa: F811
    import numpy as np
    import torch
    layers, lens = 131, [100, 37]
    pool, tables = make(H, dtype, layers, lens, 2, 64, seed=13)
    scores = torch.rand((layers, 2, 2, 100), generator=torch.Generator().manual_seed(2)).cuda()
    dev = torch.from_numpy(tables.astype(np.int32)).cuda()
    ev = H.CacheEviction(pool, dev, i32(lens), scores, 40, 5)
    before = snapshot(pool)
    assert ev.evict().tolist() == [40, 37] and int(ev.status.item()) == 0
    want = plain_compact(before, layers, 2, tables, lens, ev.kept.cpu().numpy(), [40, 37], dtype == "e4m3")
    got = snapshot(pool)
    for k in want:
        assert np.array_equal(got[k], want[k]), k
