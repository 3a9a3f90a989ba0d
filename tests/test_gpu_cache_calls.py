"""Calls of the cache operators that their documentation allows and that are easy to get wrong."""
import ctypes

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
