"""Calls of the cache operators that their documentation allows and that are easy to get wrong: handles used on another stream than they were made on,
padded batches, bounds without a limit, a call after one that failed."""
import ctypes
import gc
import sys

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


def batch(H, lens, kv_heads=2, head_dim=64, dtype="f16", seed=0, layers=1):
    """A pool of normal values, block tables in order, q, all on the device."""
    import torch
    g = torch.Generator().manual_seed(seed)
    width = max((t + BS - 1) // BS for t in lens)
    pool = H.Pool.allocate(0, layers, kv_heads, head_dim, BS, len(lens) * width, dtype)
    for layer in range(layers):
        for is_v in (False, True):
            x = torch.randn((len(lens) * width, BS, kv_heads, head_dim), generator=g)
            pool.blocks(layer, is_v).copy_(x.to(torch.float16) if dtype == "f16" else x.to(torch.float8_e4m3fn).view(torch.uint8))
    tables = torch.arange(len(lens) * width, dtype=torch.int32).view(len(lens), width).cuda()
    q = torch.randn((len(lens), kv_heads * 2, head_dim), generator=g).to(torch.float16).cuda()
    return pool, tables, q, torch.tensor(lens, dtype=torch.int32).cuda()


def test_handles_used_at_once_on_another_stream_than_they_were_made_on(H):
    """The stream on which a handle is made is busy; the call goes to another one, whose order with the caller's tensors is the caller's business but
    which cannot know of the handle's own buffers.  A first round loads the kernels and fills the allocator, so that nothing else waits."""
    import torch
    pool, tables, q, lens = batch(H, [60, 200, 33])
    i32 = lambda v: torch.tensor(v, dtype=torch.int32).cuda()  # noqa: E731
    starts, prefixes = i32([0, 3]), i32([32])
    scores, into = torch.rand((1, 3, 2, 208), generator=torch.Generator().manual_seed(1)).cuda(), torch.zeros((1, 3, 2, 208)).cuda()
    bad = tables.clone()
    bad[:, 1] = 1 << 24
    side = torch.cuda.Stream()
    for busy in (False, True):
        torch.cuda.synchronize()
        if busy:
            torch.cuda._sleep(400_000_000)                             # some 0.2 s
        ev = H.CacheEviction(None, None, lens, scores, 40, 8)
        ev.select(side)
        handles = [H.ScoredDecodeAttention(pool, q, bad, lens, into, 200), H.PrefixAttention(pool, q, bad, lens, starts, prefixes, 200, 32)]
        for h in handles:
            h.enqueue(0, side)
        torch.cuda.synchronize()
        kept, new, told = ev.kept.clone(), ev.new_lens.clone(), [int(h.status.item()) for h in handles]
        if not busy:
            want = kept, new
        del ev, handles, h
    assert torch.equal(kept, want[0]) and torch.equal(new, want[1]) and new.tolist() == [40, 40, 33]
    assert told == [N.ERR_INVALID_CONFIG] * 2                          # what the kernels reported is still there


def test_a_handle_dropped_while_its_call_runs_on_another_stream_keeps_its_workspace(H):
    import torch
    pool, tables, q, lens = batch(H, [60, 200, 33])
    i32 = lambda v: torch.tensor(v, dtype=torch.int32).cuda()  # noqa: E731
    starts, prefixes = i32([0, 3]), i32([32])
    side = torch.cuda.Stream()
    first = H.PrefixAttention(pool, q, tables, lens, starts, prefixes, 200, 32)
    want, size = first.enqueue(0).clone(), first.scratch.numel()
    h = H.PrefixAttention(pool, q, tables, lens, starts, prefixes, 200, 32)
    h.enqueue(0, side)
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        torch.cuda._sleep(200_000_000)
    out, at = h.enqueue(0, side), h.scratch.data_ptr()
    del h
    gc.collect()                                                       # (a handle refers to itself)
    again = [torch.empty(size, dtype=torch.uint8, device="cuda") for _ in range(100)]   # the allocator must not hand out what the call still uses
    assert all(x.data_ptr() >= at + size or x.data_ptr() + size <= at for x in again)
    torch.cuda.synchronize()
    assert torch.equal(out, want)


def test_lengths_of_rows_outside_the_groups_are_nobodys_business(H):
    """A padded batch: what stands in kv_lens (and the tables) behind the last group, and before the first, is not looked at."""
    import torch
    pool, tables, q, lens = batch(H, [60, 200, 33, 40, 90])
    i32 = lambda v: torch.tensor(v, dtype=torch.int32).cuda()  # noqa: E731
    starts, prefixes = i32([1, 3]), i32([0])
    attn = H.PrefixAttention(pool, q, tables, lens, starts, prefixes, 200, 16)
    want = attn.enqueue(0).clone()
    assert int(attn.status.item()) == 0
    lens[0], lens[3], lens[4] = -1, 100000, -7
    tables[3:] = -1
    attn.out.fill_(7.5)
    out = attn.enqueue(0)
    assert int(attn.status.item()) == 0
    assert torch.equal(out[1:3], want[1:3]) and (out[0] == 7.5).all() and (out[3:] == 7.5).all()


@pytest.mark.parametrize("budget,recent", [(1 << 32, 4), (sys.maxsize, 0), (4, 1 << 32), (4, sys.maxsize)])
def test_a_budget_without_a_limit_cuts_nothing(H, budget, recent):
    import torch
    scores = torch.rand((1, 2, 1, 64)).cuda()
    ev = H.CacheEviction(None, None, torch.tensor([64, 50], dtype=torch.int32).cuda(), scores, budget, recent)
    kept, new = ev.select()
    assert int(ev.status.item()) == 0 and new.tolist() == [64, 50]
    assert kept[0, 0, 0].tolist() == list(range(64))


def test_negative_budgets_are_refused(H):
    import torch
    scores, lens = torch.rand((1, 1, 1, 64)).cuda(), torch.tensor([64], dtype=torch.int32).cuda()
    for budget, recent in ((-1, 0), (8, -1)):
        with pytest.raises(H.TkvError):
            H.CacheEviction(None, None, lens, scores, budget, recent)


def test_a_call_that_fails_on_its_device_spoils_nothing_after_it(H):
    """A device that does not exist: the call says so, and neither the next call nor torch finds that error again."""
    import torch
    pool, tables, q, lens = batch(H, [60, 200, 33])
    i32 = lambda v: torch.tensor(v, dtype=torch.int32).cuda()  # noqa: E731
    scores = torch.rand((1, 3, 2, 208), generator=torch.Generator().manual_seed(1)).cuda()
    ev = H.CacheEviction(pool, tables, lens, scores, 40, 8)
    scored, pre = H.ScoredDecodeAttention(pool, q, tables, lens, scores, 200), H.PrefixAttention(pool, q, tables, lens, i32([0, 3]), i32([32]), 200, 32)
    nowhere = type(ev._pool_c).from_buffer_copy(ev._pool_c)
    nowhere.device = 1 << 20
    select = type(ev._select).from_buffer_copy(ev._select)
    select.device = 1 << 20
    L, none = N.lib(), ctypes.c_void_p(0)

    def good():
        torch.zeros(4, device="cuda").add_(1)                          # torch looks for errors after a launch
        ev.select()
        ev.compact()
        scored.enqueue(0)
        pre.enqueue(0)
    good()
    for call in (lambda: L.tkv_evict_select_enqueue(ctypes.byref(select), none),
                 lambda: L.tkv_evict_compact_enqueue(ctypes.byref(nowhere), ctypes.byref(ev._compact), none),
                 lambda: L.tkv_scored_attn_enqueue(ctypes.byref(nowhere), ctypes.byref(scored._mk(0)), none),
                 lambda: L.tkv_prefix_attn_enqueue(ctypes.byref(nowhere), ctypes.byref(pre._mk(0)), none)):
        assert call() == N.ERR_CUDA
        good()
    torch.cuda.synchronize()
    assert int(ev.status.item()) == int(scored.status.item()) == int(pre.status.item()) == 0


@pytest.mark.parametrize("dtype", ["f16", "e4m3"])
def test_a_foreign_block_deep_in_a_prefix_ends_the_call_and_leaves_the_next_one_alone(H, dtype):
    """The producer meets the id with tiles before it on their way and under the tensor cores: the call reports it and returns, again and again."""
    import torch
    i32 = lambda v: torch.tensor(v, dtype=torch.int32).cuda()  # noqa: E731
    pool, tables, q, lens = batch(H, [3200] * 4, kv_heads=4, head_dim=128, dtype=dtype, seed=5)
    tables[:, :200] = tables[0, :200]
    good = H.PrefixAttention(pool, q, tables, lens, i32([0, 4]), i32([3200]), 3200, 3200)
    want = good.enqueue(0).clone()
    for at in (0, 7, 8, 9, 23, 100, 199):
        broken = tables.clone()
        broken[0, at] = pool.total_blocks + at
        bad = H.PrefixAttention(pool, q, broken, lens, i32([0, 4]), i32([3200]), 3200, 3200)
        for _ in range(10):
            bad.enqueue(0)
            good.enqueue(0)
        assert int(bad.status.item()) == N.ERR_INVALID_CONFIG
        assert int(good.status.item()) == 0 and torch.equal(good.out, want)
