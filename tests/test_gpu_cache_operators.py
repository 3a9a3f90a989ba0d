"""The operators of a cache under a decode loop -- scored decode attention, shared-prefix attention, eviction (select and compact) --
against plain implementations in 64 bits.

Tolerances.  A weight is 2^(x - M) / L with x accumulated in F32 from exact F16 products: for |x| < 32 in the log2 domain an
error of 16 roundings (8 k-steps of the MMA in two chains, their sum, the scale, the subtraction, and as many again for the
truncating adds inside an MMA) of 2^-24 * 32 each is 3.1e-5 at the very worst, times ln 2 for the weight, plus 2^-22 of the exp2: 2.2e-5
relative; F32 q adds its own 2^-22 per element times sqrt(128) terms of random sign, below 1e-5 of |x| <= 32.  Bound used: 4e-5 of the weight
and 1e-7 of the row's largest weight.
out: an F16 probability is off by 2^-12 of itself (half a step, 2^-11 relative spacing at most 2^-11: eps / 2 = 2^-11), so out by at most
2^-11 * sum |w v| <= 2^-11 * max |v|; the weights' own 4e-5 and the final rounding to F16, 2^-11 * |out|, come on top.  With F32 q the
probabilities keep 22 bits: 4e-5 * max |v| covers all."""
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


class Cache:
    """A pool of garbage (NaN, infinities) with a batch's rows written into shuffled blocks, and its values in 64 bits."""

    def __init__(self, H, lens, kv_heads, head_dim, dtype, layers=1, seed=0, shared=None, spare=3):
        import torch
        g = torch.Generator().manual_seed(seed)
        self.lens, self.kv_heads, self.head_dim = list(lens), kv_heads, head_dim
        width = max(1, max((t + BS - 1) // BS for t in self.lens))
        rows, count, first = [], 0, {}
        for s, t in enumerate(self.lens):
            nb = (t + BS - 1) // BS
            row = []
            if shared is not None and shared[s] is not None:          # (group, prefix blocks)
                grp, pre = shared[s]
                if grp not in first:
                    first[grp] = list(range(count, count + pre))
                    count += pre
                row = first[grp][:nb]
            row = row + list(range(count, count + nb - len(row)))
            count = max([count] + [r + 1 for r in row])
            rows.append(row + [-1] * (width - nb))                    # never read: -1 is outside every pool
        total = count + spare
        perm = torch.randperm(total, generator=g)
        self.tables = torch.tensor([[int(perm[b]) if b >= 0 else -1 for b in r] for r in rows], dtype=torch.int32)
        scaled = dtype == "e4m3"
        self.pool = H.Pool.allocate(0, layers, kv_heads, head_dim, BS, total, "f16" if dtype == "f16" else "e4m3", scales=scaled, fill_byte=None)
        self.values = {}
        for layer in range(layers):
            for is_v in (False, True):
                x = torch.randn((total, BS, kv_heads, head_dim), generator=g) * 0.5
                x[..., head_dim // 3] *= 6
                x = x.to(torch.float16)
                view = self.pool.blocks(layer, is_v)
                live = torch.zeros((total, BS), dtype=torch.bool)
                for s, t in enumerate(self.lens):
                    for b in range((t + BS - 1) // BS):
                        live[int(self.tables[s, b]), : min(BS, t - b * BS)] = True
                if dtype == "f16":
                    val = x.double()
                    bad = torch.full_like(x, float("nan"))
                    bad[..., ::2] = float("inf")
                    view.copy_(torch.where(live[:, :, None, None], x, bad))
                else:
                    y, sc = x.float(), torch.ones((total, kv_heads))
                    if scaled:
                        sc = (torch.where(live[:, :, None, None], y, torch.zeros_like(y)).abs().amax(dim=(1, 3)) / 448).clamp_min(1e-6)
                        sc[::3] *= 64                               # blocks of very different scales side by side
                        y = y / sc[:, None, :, None]
                    y = torch.where(y.abs() < 2.0 ** -6, torch.zeros_like(y), y).clamp(-448, 448).to(torch.float8_e4m3fn)
                    val = y.float().double() * sc.double()[:, None, :, None]
                    raw = torch.where(live[:, :, None, None], y.view(torch.uint8), torch.full(y.shape, 0x7F, dtype=torch.uint8))   # NaN bytes
                    view.copy_(raw)
                    if scaled:
                        (self.pool.v_scales if is_v else self.pool.k_scales)[layer].copy_(sc)
                self.values[layer, is_v] = val
        self.dev_tables = self.tables.cuda()
        self.dev_lens = torch.tensor(self.lens, dtype=torch.int32).cuda()
        torch.cuda.synchronize()

    def rows(self, layer, is_v, s, n=None):
        """[tokens, kv_heads, head_dim] of sequence s in 64 bits."""
        n = self.lens[s] if n is None else n
        blocks = self.tables[s, : (n + BS - 1) // BS].long()
        return self.values[layer, is_v][blocks].flatten(0, 1)[:n]

    def attention(self, layer, q, scale):
        """Per sequence: (out [heads, dim], weights [heads, tokens], max |v| per kv head)."""
        import torch
        res = []
        hq = q.shape[1]
        grp = hq // self.kv_heads
        for s in range(len(self.lens)):
            if self.lens[s] == 0:
                res.append((torch.zeros(hq, self.head_dim, dtype=torch.float64), torch.zeros(hq, 0, dtype=torch.float64), torch.zeros(hq, 1, dtype=torch.float64)))
                continue
            k = self.rows(layer, False, s).repeat_interleave(grp, dim=1)
            v = self.rows(layer, True, s).repeat_interleave(grp, dim=1)
            x = torch.einsum("hd,thd->ht", q[s].double(), k) * scale
            w = torch.softmax(x, dim=1)
            res.append((torch.einsum("ht,thd->hd", w, v), w, v.abs().amax(dim=(0, 2))[:, None]))
        return res


def out_close(got, want, vmax, f32):
    import torch
    got = got.double().cpu()
    bound = (4e-5 if f32 else 2.0 ** -11 + 4e-5) * vmax + (2.0 ** -23 if f32 else 2.0 ** -11) * want.abs() + 1e-7
    err = (got - want).abs()
    assert torch.isfinite(got).all()
    assert (err <= bound).all(), f"off by {(err / bound).max():.2f} of the bound"


def scores_close(got, want, start):
    """got, want: after the step; `start`: before it."""
    import torch
    got = got.double().cpu()
    w = want - start
    bound = 4e-5 * w.abs() + 2.0 ** -22 * want.abs() + 1e-7 * w.abs().max().clamp_min(0)
    err = (got - want).abs()
    assert (err <= bound).all(), f"off by {(err / bound.clamp_min(1e-30)).max():.2f} of the bound"


# ---- scored decode attention ----------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", ["f16", "e4m3", "e4m3 unscaled"])
@pytest.mark.parametrize("kv_heads,head_dim,group", [(8, 128, 4), (4, 64, 8), (1, 128, 1), (5, 128, 3), (3, 64, 2), (16, 64, 1), (2, 128, 8)])
@pytest.mark.parametrize("f32", [False, True])
def test_scored_attention(H, dtype, kv_heads, head_dim, group, f32):
    import torch
    lens = [1, 15, 0, 16, 17, 63, 64, 65, 400, 1029, 33, 0]
    c = Cache(H, lens, kv_heads, head_dim, dtype, layers=2, seed=kv_heads * 7 + head_dim)
    g = torch.Generator().manual_seed(5)
    q = torch.randn((len(lens), kv_heads * group, head_dim), generator=g) * 2
    q = q if f32 else q.to(torch.float16)
    stride = max(lens) + 3
    start = torch.rand((2, len(lens), kv_heads, stride), generator=g)
    for s, t in enumerate(lens):
        start[:, s, :, t:] = float("nan")                            # behind the end: never read, never written
    scores = start.cuda()
    decay = 0.75
    attn = H.ScoredDecodeAttention(c.pool, q.cuda(), c.dev_tables, c.dev_lens, scores, max(lens), decay=decay)
    for layer in (1, 0):
        out = attn.enqueue(layer).clone()
        assert int(attn.status.item()) == 0
        for s, (want, w, vmax) in enumerate(c.attention(layer, q, attn.sm_scale)):
            out_close(out[s], want, vmax, f32)
            t = lens[s]
            if t:
                before = start[layer, s, :, :t].double() * decay
                scores_close(scores[layer, s, :, :t], before + w.view(kv_heads, group, t).sum(dim=1), before)
    assert torch.equal(torch.isnan(scores).cpu(), torch.isnan(start))


def test_scored_attention_long_context_overwrites_at_decay_zero(H):
    """One sequence split over the whole grid, its scores starting as NaN: decay 0 does not read them.  The weights of a row sum to the group."""
    import torch
    n = 20011
    c = Cache(H, [n], 2, 128, "f16", seed=3)
    q = (torch.randn((1, 16, 128), generator=torch.Generator().manual_seed(1)) * 2).to(torch.float16)
    scores = torch.full((1, 1, 2, n), float("nan")).cuda()
    attn = H.ScoredDecodeAttention(c.pool, q.cuda(), c.dev_tables, c.dev_lens, scores, n, decay=0.0)
    out = attn.enqueue(0)
    (want, w, vmax), = c.attention(0, q, attn.sm_scale)
    out_close(out[0], want, vmax, False)
    w = w.view(2, 8, n).sum(dim=1)
    scores_close(scores[0, 0], w, torch.zeros_like(w))
    assert abs(float(scores.double().sum()) - 16.0) < 16 * 1e-5
    again = scores.clone()
    attn.enqueue(0)
    assert torch.equal(scores, again)                                 # no atomics: the same bits every time


def test_scored_attention_more_sequences_than_a_cta_caches(H):
    """1 500 sequences of 0 to 40 tokens: more than a CTA keeps the ranges of, several to one share, many empty."""
    import torch
    lens = [(s * 7919) % 41 if s % 3 else 0 for s in range(1500)]
    c = Cache(H, lens, 2, 64, "f16", seed=4)
    q = torch.randn((1500, 4, 64), generator=torch.Generator().manual_seed(2)).to(torch.float16)
    scores = torch.zeros((1, 1500, 2, 48)).cuda()
    attn = H.ScoredDecodeAttention(c.pool, q.cuda(), c.dev_tables, c.dev_lens, scores, 48)
    out = attn.enqueue(0)
    assert int(attn.status.item()) == 0
    for s, (want, w, vmax) in enumerate(c.attention(0, q, attn.sm_scale)):
        out_close(out[s], want, vmax, False)
        if lens[s]:
            w = w.view(2, 2, lens[s]).sum(dim=1)
            scores_close(scores[0, s, :, : lens[s]], w, torch.zeros_like(w))
    for s, t in enumerate(lens):
        assert (scores[0, s, :, t:] == 0).all()


def test_scored_attention_in_a_graph_and_on_another_stream(H):
    """Captured once, replayed after lengths, q and scores changed in place; a call on another stream than the tensors' own."""
    import torch
    lens = [70, 200]
    c = Cache(H, lens, 4, 64, "e4m3", seed=6)
    q = torch.randn((2, 32, 64), generator=torch.Generator().manual_seed(9)).to(torch.float16)
    dq, scores = q.cuda(), torch.zeros((1, 2, 4, 256)).cuda()
    attn = H.ScoredDecodeAttention(c.pool, dq, c.dev_tables, c.dev_lens, scores, 256 - 48)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        attn.enqueue(0)
    torch.cuda.current_stream().wait_stream(side)
    first, first_scores = attn.out.clone(), scores.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        attn.enqueue(0)
    scores.zero_()
    graph.replay()
    assert torch.equal(attn.out, first) and torch.equal(scores, first_scores)
    c.dev_lens.copy_(torch.tensor([33, 0], dtype=torch.int32))
    c.lens = [33, 0]
    scores.zero_()
    graph.replay()
    (want, w, vmax), (zero, _, _) = c.attention(0, q, attn.sm_scale)
    out_close(attn.out[0], want, vmax, False)
    assert (attn.out[1] == 0).all()
    assert (scores[0, 1] == 0).all() and (scores[0, 0, :, 33:] == 0).all()


def test_scored_attention_reports_bad_lengths_and_blocks(H):
    import torch
    c = Cache(H, [40, 90], 2, 64, "f16", seed=8)
    q = torch.randn((2, 4, 64)).to(torch.float16).cuda()
    scores = torch.zeros((1, 2, 2, 128)).cuda()
    attn = H.ScoredDecodeAttention(c.pool, q, c.dev_tables, torch.tensor([40, 100000], dtype=torch.int32).cuda(), scores, 90)
    attn.enqueue(0)
    assert int(attn.status.item()) == N.ERR_INVALID_CONFIG
    assert (scores[0, 1, :, 90:] == 0).all()                           # clamped
    bad = c.dev_tables.clone()
    bad[1, 2] = 1 << 20
    attn = H.ScoredDecodeAttention(c.pool, q, bad, c.dev_lens, scores, 90)
    attn.enqueue(0)
    assert int(attn.status.item()) == N.ERR_INVALID_CONFIG


def test_scored_attention_masked_rows_and_extreme_scores(H):
    """Scores of +-6e4 (far outside exp's range) and equal scores: the maximum is subtracted, ties share."""
    import torch
    c = Cache(H, [50], 1, 64, "f16", seed=2)
    c.pool.blocks(0, False).zero_()
    k = torch.zeros((50, 64), dtype=torch.float16)
    k[:, 0] = torch.linspace(-200, 200, 50).to(torch.float16)
    k[30:, 0] = 200.0
    for t in range(50):
        c.pool.blocks(0, False)[int(c.tables[0, t // BS]), t % BS, 0] = k[t].cuda()
    q = torch.zeros((1, 2, 64), dtype=torch.float16)
    q[0, 0, 0] = 300.0
    scores = torch.zeros((1, 1, 1, 64)).cuda()
    attn = H.ScoredDecodeAttention(c.pool, q.cuda(), c.dev_tables, c.dev_lens, scores, 50, sm_scale=1.0)
    out = attn.enqueue(0).double().cpu()
    v = c.rows(0, True, 0)[:, 0]
    assert torch.allclose(out[0, 0], v[30:].mean(dim=0), atol=2e-3)    # head 0: the twenty equal maxima
    assert torch.allclose(out[0, 1], v.mean(dim=0), atol=2e-3)         # head 1: q = 0, all tokens alike
    want = torch.full((50,), 1 / 50, dtype=torch.float64)
    want[30:] += 1 / 20
    assert torch.allclose(scores[0, 0, 0, :50].double().cpu(), want, rtol=1e-6)


def test_scored_attention_refusals(H):
    import torch
    c = Cache(H, [40], 2, 64, "f16", seed=1)
    q = torch.zeros((1, 4, 64), dtype=torch.float16).cuda()
    scores = torch.zeros((1, 1, 2, 64)).cuda()

    def code(change, **kw):
        attn = H.ScoredDecodeAttention(c.pool, q, c.dev_tables, c.dev_lens, scores, 40, **kw)
        args = attn._mk(0)
        for name, value in change.items():
            setattr(args, name, value)
        import ctypes
        rc = N.lib().tkv_scored_attn_enqueue(ctypes.byref(attn._pool_c), ctypes.byref(args), None)
        return rc
    assert code({}) == 0
    assert code({"n_seqs": 0}) == 0
    for change in ({"layer": 1}, {"q": 0}, {"out": 0}, {"tables": 0}, {"kv_lens": 0}, {"scores": 0}, {"q_dtype": N.DTYPE_E4M3}, {"decay": 1.5},
                   {"decay": float("nan")}, {"sm_scale": float("inf")}, {"q": q.data_ptr() + 2}, {"scores": scores.data_ptr() + 2}):
        assert code(change) == N.ERR_INVALID_CONFIG, change
    for change in ({"n_q_heads": 3}, {"n_q_heads": 18}, {"table_stride": 2}, {"score_stride": 39}, {"scratch_bytes": 100}, {"scratch": 0}):
        assert code(change) == N.ERR_DIMENSION_MISMATCH, change


@pytest.mark.parametrize("dtype,kv_heads,head_dim,group", [("f16", 8, 128, 4), ("e4m3", 8, 128, 4), ("e4m3", 7, 128, 2), ("f16", 2, 64, 8), ("e4m3", 1, 64, 4)])
def test_scored_attention_long_shares(H, dtype, kv_heads, head_dim, group):
    """Enough blocks that every part walks its ring many times round, across sequences."""
    import torch
    lens = [3000 + 531 * s for s in range(9)] + [1, 17]
    c = Cache(H, lens, kv_heads, head_dim, dtype, seed=11)
    q = (torch.randn((len(lens), kv_heads * group, head_dim), generator=torch.Generator().manual_seed(3)) * 2).to(torch.float16)
    scores = torch.zeros((1, len(lens), kv_heads, max(lens))).cuda()
    attn = H.ScoredDecodeAttention(c.pool, q.cuda(), c.dev_tables, c.dev_lens, scores, max(lens))
    for rep in range(20):                                            # back to back over one workspace
        if rep == 19:
            scores.zero_()
        out = attn.enqueue(0)
    assert int(attn.status.item()) == 0
    for s, (want, w, vmax) in enumerate(c.attention(0, q, attn.sm_scale)):
        out_close(out[s], want, vmax, False)
        w = w.view(kv_heads, group, lens[s]).sum(dim=1)
        scores_close(scores[0, s, :, : lens[s]], w, torch.zeros_like(w))


# ---- shared-prefix attention --------------------------------------------------------------------------------------------------------
def grouped(sizes, prefixes, suffixes):
    """(starts, prefix lengths, per-sequence (group, prefix blocks), lengths) of a batch; suffixes go round."""
    starts, shared, lens = [0], [], []
    for g, (n, p) in enumerate(zip(sizes, prefixes)):
        for i in range(n):
            shared.append((g, p // BS))
            lens.append(max(0, p + suffixes[len(lens) % len(suffixes)]))
        starts.append(starts[-1] + n)
    return starts, shared, lens


def prefix_case(H, dtype, kv_heads, head_dim, group, sizes, prefixes, suffixes, seed=0, pad=0, gain=2.0):
    import torch
    starts, shared, lens = grouped(sizes, prefixes, suffixes)
    c = Cache(H, lens + [40] * pad, kv_heads, head_dim, dtype, layers=1, seed=seed, shared=shared + [None] * pad)
    n = len(lens) + pad
    q = (torch.randn((n, kv_heads * group, head_dim), generator=torch.Generator().manual_seed(seed + 1)) * gain).to(torch.float16)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32).cuda()  # noqa: E731
    width = max(c.tables.shape[1], max(prefixes) // BS)
    tables = torch.full((n, width), -1, dtype=torch.int32)
    tables[:, : c.tables.shape[1]] = c.tables
    first = {}
    for s, (g, blocks) in enumerate(shared):                          # a group's first row names the whole prefix, however short the member
        first.setdefault(g, s)
        longest = max((t for t in range(n - pad) if shared[t][0] == g), key=lambda t: lens[t])
        if s == first[g]:
            tables[s, :blocks] = c.tables[longest, :blocks]
    attn = H.PrefixAttention(c.pool, q.cuda(), tables.cuda(), c.dev_lens, i32(starts), i32(prefixes), max(lens + [40]), max(prefixes))
    return c, q, attn, lens


@pytest.mark.parametrize("dtype", ["f16", "e4m3", "e4m3 unscaled"])
@pytest.mark.parametrize("kv_heads,head_dim,group", [(8, 128, 4), (4, 64, 8), (1, 128, 1), (5, 128, 3), (3, 64, 2), (2, 128, 8), (2, 64, 7)])
@pytest.mark.parametrize("sizes,prefixes,suffixes", [
    ([3], [48], [1, 20, 5]),                                          # one short tile
    ([1, 5, 2, 40], [16, 400, 0, 1040], [0, 7, 33, 100, 1]),          # uneven groups, one without a prefix, sequences with nothing of their own
    ([70], [272], [17, 0, 3]),                                        # several row blocks for larger groups of heads
    ([2, 2], [128, 256], [16, 64]),                                   # whole tiles
])
def test_prefix_attention(H, dtype, kv_heads, head_dim, group, sizes, prefixes, suffixes):
    import torch
    c, q, attn, lens = prefix_case(H, dtype, kv_heads, head_dim, group, sizes, prefixes, suffixes, seed=kv_heads + head_dim + len(sizes))
    attn.out.fill_(float("nan"))
    out = attn.enqueue(0)
    assert int(attn.status.item()) == 0
    for s, (want, _, vmax) in enumerate(c.attention(0, q, attn.sm_scale)):
        out_close(out[s], want, vmax, False)
    again = out.clone()
    attn.enqueue(0)
    assert torch.equal(attn.out, again)                               # no atomics: the same bits every time


@pytest.mark.parametrize("dtype", ["f16", "e4m3"])
def test_prefix_attention_long_prefix(H, dtype):
    """More cached tiles than CTAs, shares that begin and end inside items, two row blocks of which the second is short."""
    c, q, attn, lens = prefix_case(H, dtype, 2, 128, 8, [40, 3], [9008, 4096], [40, 0, 100], seed=3)
    out = attn.enqueue(0)
    assert int(attn.status.item()) == 0
    for s, (want, _, vmax) in enumerate(c.attention(0, q, attn.sm_scale)):
        out_close(out[s], want, vmax, False)


def test_prefix_attention_leaves_padded_rows_and_serves_short_members(H):
    """Rows behind the last group stay as they were; a member shorter than its group's prefix, or empty, gets its own tokens only."""
    import torch
    starts, shared, lens = grouped([4], [64], [10])
    lens = [74, 40, 0, 64]
    c = Cache(H, lens + [40, 40], 2, 64, "f16", seed=4, shared=shared + [None, None])
    q = torch.randn((6, 8, 64), generator=torch.Generator().manual_seed(1)).to(torch.float16)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32).cuda()  # noqa: E731
    attn = H.PrefixAttention(c.pool, q.cuda(), c.dev_tables, c.dev_lens, i32([0, 4]), i32([64]), 74, 64)
    attn.out.fill_(7.5)
    out = attn.enqueue(0)
    assert int(attn.status.item()) == 0
    assert (out[4:] == 7.5).all()
    for s, (want, _, vmax) in enumerate(c.attention(0, q, attn.sm_scale)[:4]):
        out_close(out[s], want, vmax, False)
    assert (out[2] == 0).all()


@pytest.mark.parametrize("dtype", ["f16", "e4m3"])
@pytest.mark.parametrize("head_dim", [64, 128])
def test_prefix_attention_row_blocks_of_every_width(H, dtype, head_dim):
    """Groups of one query head per kv head whose row counts are at, below and above each width at which rows are laid out differently."""
    sizes = [1, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 256, 257]
    c, q, attn, lens = prefix_case(H, dtype, 1, head_dim, 1, sizes, [16 * (1 + 3 * g) for g in range(len(sizes))], [3, 0, 17], seed=21)
    attn.out.fill_(float("nan"))
    out = attn.enqueue(0)
    assert int(attn.status.item()) == 0
    for s, (want, _, vmax) in enumerate(c.attention(0, q, attn.sm_scale)):
        out_close(out[s], want, vmax, False)


@pytest.mark.parametrize("dtype", ["f16", "e4m3"])
@pytest.mark.parametrize("poison", ["nan", "inf"])
def test_prefix_attention_member_shorter_than_its_prefix_sees_nothing_behind_its_end(H, dtype, poison):
    """What the prefix holds behind a short member's end, NaN and infinities included, is no part of that member's result."""
    import torch
    c, q, attn, lens = prefix_case(H, dtype, 2, 128, 4, [3, 2], [160, 32], [-90, 5, 0, -16, 3], seed=22)
    assert lens[0] == 70 and lens[3] == 16
    for s, first in ((0, 70), (3, 16)):
        for t in range(first, 160 if s == 0 else 32):
            for is_v in (False, True):
                row = c.pool.blocks(0, is_v)[int(attn.tables[s, t // BS]), t % BS]
                if dtype == "f16":
                    row.fill_(float(poison) * (-1 if t % 2 else 1))
                else:
                    row.fill_(0x7F if t % 2 else 0xFF)                # the type has no infinity
    attn.out.fill_(float("nan"))
    out = attn.enqueue(0)
    assert int(attn.status.item()) == 0
    want = c.attention(0, q, attn.sm_scale)
    for s in (0, 3):
        out_close(out[s], want[s][0], want[s][2], False)


def test_prefix_attention_equals_decode_attention_without_groups_of_more_than_one(H):
    """Every sequence its own group: what the plain decode attention computes, to both kernels' rounding."""
    import torch
    c, q, attn, lens = prefix_case(H, "f16", 8, 128, 4, [1] * 9, [16 * (s % 5) for s in range(9)], [30, 5], seed=6)
    out = attn.enqueue(0).float()
    ref = H.decode_attention(c.pool, 0, q.float().cuda(), c.dev_tables, c.dev_lens)
    for s, (want, _, vmax) in enumerate(c.attention(0, q, attn.sm_scale)):
        out_close(out[s], want, vmax, False)
    assert (out - ref).abs().max() < 2e-2


def test_prefix_attention_in_a_graph_with_changing_groups(H):
    """Captured once; lengths, groups and prefixes change in place between replays."""
    import torch
    c, q, attn, lens = prefix_case(H, "f16", 4, 64, 4, [3, 4], [96, 64], [20, 9], seed=8)
    attn.enqueue(0)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        attn.enqueue(0)
    attn.out.zero_()
    graph.replay()
    for s, (want, _, vmax) in enumerate(c.attention(0, q, attn.sm_scale)):
        out_close(attn.out[s], want, vmax, False)
    attn.prefix_lens.copy_(torch.tensor([48, 0], dtype=torch.int32))  # a shorter shared part is as right
    attn.group_starts.copy_(torch.tensor([0, 3, 6], dtype=torch.int32))
    attn.out.fill_(3.0)
    graph.replay()
    for s, (want, _, vmax) in enumerate(c.attention(0, q, attn.sm_scale)[:6]):
        out_close(attn.out[s], want, vmax, False)
    assert (attn.out[6] == 3.0).all()


def test_two_calls_at_once_on_two_streams(H):
    """Handles of their own share no workspace: calls that run side by side give what each gives alone, bit for bit."""
    import torch
    cases = [prefix_case(H, "f16", 2, 64, 4, [5, 40], [400, 1600], [20, 3], seed=31), prefix_case(H, "e4m3", 4, 128, 2, [9, 1], [320, 64], [70], seed=32)]
    alone = [attn.enqueue(0).clone() for _, _, attn, _ in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    for _ in range(20):
        for (_, _, attn, _), stream in zip(cases, streams):
            with torch.cuda.stream(stream):
                attn.out.fill_(float("nan"))
            attn.enqueue(0, stream)
    torch.cuda.synchronize()
    for (_, _, attn, _), want in zip(cases, alone):
        assert int(attn.status.item()) == 0
        assert torch.equal(attn.out, want)


def test_prefix_attention_negative_scale_and_equal_scores(H):
    import torch
    c, q, attn, lens = prefix_case(H, "f16", 2, 64, 2, [3], [160], [5], seed=9)
    neg = H.PrefixAttention(c.pool, attn.q, attn.tables, attn.kv_lens, attn.group_starts, attn.prefix_lens, max(lens), 160, sm_scale=-0.2)
    out = neg.enqueue(0)
    for s, (want, _, vmax) in enumerate(c.attention(0, q, -0.2)):
        out_close(out[s], want, vmax, False)
    flat = H.PrefixAttention(c.pool, attn.q, attn.tables, attn.kv_lens, attn.group_starts, attn.prefix_lens, max(lens), 160, sm_scale=0.0)
    out = flat.enqueue(0)
    for s, (want, _, vmax) in enumerate(c.attention(0, q, 0.0)):
        out_close(out[s], want, vmax, False)


def test_prefix_attention_reports_what_it_cannot_trust(H):
    import torch
    c, q, attn, lens = prefix_case(H, "f16", 2, 64, 2, [2, 2], [64, 32], [9], seed=10)
    good = attn.enqueue(0).clone()
    i32 = lambda v: torch.tensor(v, dtype=torch.int32).cuda()  # noqa: E731

    def run(**kw):
        args = dict(tables=attn.tables, kv_lens=attn.kv_lens, group_starts=attn.group_starts, prefix_lens=attn.prefix_lens)
        args.update(kw)
        a = H.PrefixAttention(c.pool, attn.q, args["tables"], args["kv_lens"], args["group_starts"], args["prefix_lens"], max(lens), 64)
        a.out.fill_(5.0)
        a.enqueue(0)
        return int(a.status.item()), a.out
    assert run()[0] == 0
    for kw in ({"group_starts": i32([0, 3, 2])}, {"group_starts": i32([0, 2, 5])}, {"prefix_lens": i32([64, 40])}, {"prefix_lens": i32([80, 32])}):
        code, out = run(**kw)
        assert code == N.ERR_INVALID_CONFIG and (out == 5.0).all(), kw     # nothing is computed
    bad = attn.tables.clone()
    bad[0, 1] = 1 << 24                                                # a prefix block outside the pool
    assert run(tables=bad)[0] == N.ERR_INVALID_CONFIG
    bad = attn.tables.clone()
    bad[3, 2] = -5                                                     # one behind the prefix
    assert run(tables=bad)[0] == N.ERR_INVALID_CONFIG
    code, out = run(kv_lens=i32([lens[0], 100000, lens[2], lens[3]]))
    assert code == N.ERR_INVALID_CONFIG
    assert torch.equal(run()[1], good)                                 # the context is still usable


def test_prefix_attention_refusals(H):
    import ctypes
    c, q, attn, lens = prefix_case(H, "f16", 2, 64, 2, [2], [32], [9], seed=11)

    def code(change):
        args = attn._mk(0)
        for name, value in change.items():
            setattr(args, name, value)
        return N.lib().tkv_prefix_attn_enqueue(ctypes.byref(attn._pool_c), ctypes.byref(args), None)
    assert code({}) == 0 and code({"n_seqs": 0}) == 0 and code({"n_groups": 0}) == 0
    for change in ({"layer": 1}, {"q": 0}, {"out": 0}, {"tables": 0}, {"kv_lens": 0}, {"group_starts": 0}, {"prefix_lens": 0},
                   {"sm_scale": float("nan")}, {"q": attn.q.data_ptr() + 8}, {"scratch": attn.scratch.data_ptr() + 16}):
        assert code(change) == N.ERR_INVALID_CONFIG, change
    for change in ({"n_q_heads": 3}, {"n_q_heads": 18}, {"table_stride": 2}, {"max_prefix_len": 64}, {"scratch_bytes": 100}, {"scratch": 0}):
        assert code(change) == N.ERR_DIMENSION_MISMATCH, change
