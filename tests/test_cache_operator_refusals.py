"""The refusals of the cache operators (shared-prefix attention, scored attention, eviction) need no GPU: every argument is checked before
the first CUDA call, so made-up addresses are never followed."""
import ctypes as C

import pytest

from tempura_b200 import _build
from tempura_b200 import _native as N


@pytest.fixture(scope="module")
def L():
    _build.build()
    return N.lib()


A = 0x7F0000000000                                                     # an address that is aligned and never used


def pool(**kw):
    d = dict(device=0, dtype=N.DTYPE_F16, n_layers=2, n_kv_heads=4, head_dim=64, block_size=16, total_blocks=100, scales=0)
    d.update(kw)
    ptrs = (C.c_uint64 * max(1, d["n_layers"]))(*[A + 0x1000 * i for i in range(max(1, d["n_layers"]))])
    p = N.TkvPool(d["device"], d["dtype"], d["n_layers"], d["n_kv_heads"], d["head_dim"], d["block_size"], d["total_blocks"], 0, ptrs, ptrs,
                  d["scales"], d.get("v_scales", d["scales"]), 0)
    p._keep = ptrs
    return p


def scored(**kw):
    d = dict(n_seqs=2, n_q_heads=8, table_stride=10, layer=0, max_kv_len=160, score_stride=160, sm_scale=0.1, decay=1.0, q_dtype=N.DTYPE_F16, reserved=0,
             q=A, out=A, tables=A, kv_lens=A, scores=A, scratch=A, scratch_bytes=1 << 40, status=0)
    d.update(kw)
    return N.TkvScoredAttn(*d.values())


def prefix(**kw):
    d = dict(n_seqs=2, n_groups=1, n_q_heads=8, table_stride=10, layer=0, max_kv_len=160, max_prefix_len=64, sm_scale=0.1, q=A, out=A, tables=A, kv_lens=A,
             group_starts=A, prefix_lens=A, scratch=A, scratch_bytes=1 << 40, status=0)
    d.update(kw)
    return N.TkvPrefixAttn(*d.values())


def select(**kw):
    d = dict(device=0, n_layers=2, n_seqs=2, n_kv_heads=4, max_kv_len=160, score_stride=160, kept_stride=40, budget=40, recent=8, reserved=0, scores=A,
             kv_lens=A, protect=0, kept=A, new_lens=A, status=0)
    d.update(kw)
    return N.TkvEvictSelect(*d.values())


def compact(**kw):
    d = dict(layer_begin=0, n_layers=2, n_seqs=2, table_stride=10, max_kv_len=160, score_stride=160, kept_stride=40, reserved=0, tables=A, kv_lens=A, kept=A,
             new_lens=A, scores=0, status=0)
    d.update(kw)
    return N.TkvEvictCompact(*d.values())


BAD, DIM = N.ERR_INVALID_CONFIG, N.ERR_DIMENSION_MISMATCH
POOLS = [({"dtype": N.DTYPE_F32}, BAD), ({"head_dim": 96}, DIM), ({"block_size": 32}, DIM), ({"scales": A}, BAD),
         ({"dtype": N.DTYPE_E4M3, "scales": A, "v_scales": 0}, BAD)]


@pytest.mark.parametrize("change,code", POOLS + [({"n_kv_heads": 0}, DIM), ({"n_kv_heads": 3}, DIM), ({"total_blocks": 0}, BAD)])
def test_pools_that_attention_refuses(L, change, code):
    p = pool(**change)
    assert L.tkv_scored_attn_enqueue(C.byref(p), C.byref(scored()), None) == code
    assert L.tkv_prefix_attn_enqueue(C.byref(p), C.byref(prefix()), None) == code


@pytest.mark.parametrize("change,code", POOLS)
def test_pools_that_eviction_refuses(L, change, code):
    assert L.tkv_evict_compact_enqueue(C.byref(pool(**change)), C.byref(compact()), None) == code


@pytest.mark.parametrize("change,code", [
    ({"layer": 2}, BAD), ({"n_q_heads": 6}, DIM), ({"n_q_heads": 36}, DIM), ({"n_q_heads": 0}, DIM), ({"table_stride": 9}, DIM), ({"score_stride": 159}, DIM),
    ({"max_kv_len": 0xFFFFFFFF, "table_stride": 1 << 30}, BAD), ({"n_seqs": 0x80000000}, BAD), ({"sm_scale": float("inf")}, BAD), ({"sm_scale": float("nan")}, BAD),
    ({"decay": -0.1}, BAD), ({"decay": 1.01}, BAD), ({"decay": float("nan")}, BAD), ({"q_dtype": N.DTYPE_E4M3}, BAD), ({"q_dtype": 77}, BAD), ({"q": 0}, BAD),
    ({"out": 0}, BAD), ({"tables": 0}, BAD), ({"kv_lens": 0}, BAD), ({"scores": 0}, BAD), ({"q": A + 8}, BAD), ({"out": A + 4}, BAD), ({"scores": A + 1}, BAD),
    ({"scratch": A + 128}, BAD), ({"scratch": 0}, DIM), ({"scratch_bytes": 64}, DIM), ({"status": A + 2}, BAD)])
def test_scored_attention_refuses(L, change, code):
    assert L.tkv_scored_attn_enqueue(C.byref(pool()), C.byref(scored(**change)), None) == code


@pytest.mark.parametrize("change,code", [
    ({"layer": 2}, BAD), ({"n_q_heads": 6}, DIM), ({"n_q_heads": 36}, DIM), ({"table_stride": 9}, DIM), ({"max_prefix_len": 176}, DIM),
    ({"max_kv_len": 0xFFFFFFFF, "table_stride": 1 << 30}, BAD), ({"n_seqs": 0x80000000}, BAD), ({"sm_scale": float("inf")}, BAD), ({"q": 0}, BAD), ({"out": 0}, BAD),
    ({"tables": 0}, BAD), ({"kv_lens": 0}, BAD), ({"group_starts": 0}, BAD), ({"prefix_lens": 0}, BAD), ({"q": A + 8}, BAD), ({"scratch": A + 128}, BAD),
    ({"scratch": 0}, DIM), ({"scratch_bytes": 64}, DIM), ({"kv_lens": A + 2}, BAD)])
def test_prefix_attention_refuses(L, change, code):
    assert L.tkv_prefix_attn_enqueue(C.byref(pool()), C.byref(prefix(**change)), None) == code


def test_prefix_attention_refuses_an_f16_pool_whose_tokens_pass_31_bits(L):
    assert L.tkv_prefix_attn_enqueue(C.byref(pool(total_blocks=1 << 27)), C.byref(prefix()), None) == BAD


@pytest.mark.parametrize("change,code", [({"score_stride": 159}, DIM), ({"kept_stride": 39}, DIM), ({"recent": 41}, DIM), ({"scores": 0}, BAD), ({"kv_lens": 0}, BAD),
                                         ({"kept": 0}, BAD), ({"new_lens": 0}, BAD), ({"scores": A + 2}, BAD), ({"protect": A + 1}, BAD),
                                         ({"n_layers": 1 << 20, "n_seqs": 1 << 12}, BAD)])
def test_select_refuses(L, change, code):
    assert L.tkv_evict_select_enqueue(C.byref(select(**change)), None) == code


def test_select_refuses_to_write_the_lengths_it_reads(L):
    assert L.tkv_evict_select_enqueue(C.byref(select(kv_lens=A, new_lens=A)), None) == BAD
    text = C.create_string_buffer(256)
    L.tkv_last_error(text, 256)
    assert b"new_lens" in text.value


@pytest.mark.parametrize("change,code", [({"layer_begin": 1}, BAD), ({"n_layers": 3}, BAD), ({"layer_begin": 0xFFFFFFFF}, BAD), ({"tables": 0}, BAD), ({"kv_lens": 0}, BAD),
                                         ({"kept": 0}, BAD), ({"new_lens": 0}, BAD), ({"kept": A + 2}, BAD), ({"table_stride": 9}, DIM),
                                         ({"scores": A, "score_stride": 100}, DIM), ({"n_seqs": 0x80000000}, BAD)])
def test_compact_refuses(L, change, code):
    assert L.tkv_evict_compact_enqueue(C.byref(pool()), C.byref(compact(**change)), None) == code


def test_empty_calls_do_nothing_and_missing_arguments_are_refused(L):
    p = pool()
    assert L.tkv_scored_attn_enqueue(C.byref(p), C.byref(scored(n_seqs=0)), None) == 0
    assert L.tkv_prefix_attn_enqueue(C.byref(p), C.byref(prefix(n_seqs=0)), None) == 0
    assert L.tkv_prefix_attn_enqueue(C.byref(p), C.byref(prefix(n_groups=0)), None) == 0
    assert L.tkv_evict_select_enqueue(C.byref(select(n_seqs=0)), None) == 0
    assert L.tkv_evict_compact_enqueue(C.byref(p), C.byref(compact(n_layers=0)), None) == 0
    assert L.tkv_scored_attn_enqueue(None, C.byref(scored()), None) == BAD and L.tkv_scored_attn_enqueue(C.byref(p), None, None) == BAD
    assert L.tkv_prefix_attn_enqueue(None, C.byref(prefix()), None) == BAD and L.tkv_prefix_attn_enqueue(C.byref(p), None, None) == BAD
    assert L.tkv_evict_select_enqueue(None, None) == BAD
    assert L.tkv_evict_compact_enqueue(None, C.byref(compact()), None) == BAD and L.tkv_evict_compact_enqueue(C.byref(p), None, None) == BAD


def test_workspaces_grow_with_what_they_hold(L):
    s = L.tkv_scored_attn_scratch_bytes
    assert s(0, 8, 4, 64, 100) == 0 and s(1, 8, 0, 64, 100) == 0
    assert 0 < s(1, 8, 4, 64, 0) <= s(1, 8, 4, 64, 1) < s(1, 8, 4, 64, 5000) < s(2, 8, 4, 64, 5000) < s(2, 16, 4, 64, 5000) < s(2, 16, 4, 128, 5000)
    assert s(4096, 64, 8, 128, 131072) > 4096 * 64 * 131072 * 4           # the scores alone: past 32 bits
    p = L.tkv_prefix_attn_scratch_bytes
    assert p(0, 1, 8, 4, 64, 100, 64) == 0 and p(1, 0, 8, 4, 64, 100, 64) == 0
    assert 0 < p(1, 1, 8, 4, 64, 0, 0) <= p(1, 1, 8, 4, 64, 1000, 512) < p(64, 1, 8, 4, 64, 1000, 512) < p(64, 1, 8, 4, 128, 1000, 512)


@pytest.mark.parametrize("change", [{"protect": A + 4096}, {"protect": A + 4096 + 4}, {"protect": A + 4096 - 4}, {"kv_lens": A + 4096 + 4}, {"kv_lens": A + 4096 - 4}])
def test_select_refuses_new_lens_that_share_memory_with_what_every_row_reads(L, change):
    assert L.tkv_evict_select_enqueue(C.byref(select(new_lens=A + 4096, **change)), None) == BAD
    text = C.create_string_buffer(256)
    L.tkv_last_error(text, 256)
    assert b"new_lens" in text.value


def test_select_takes_neighbouring_buffers(L):
    """Side by side in one allocation is no overlap: the call goes on to the device (or, without one, to its error)."""
    for change in ({"protect": A + 4096 + 8}, {"protect": A + 4096 - 8}, {"kv_lens": A + 4096 + 8}, {"kv_lens": A + 4096 - 8}):
        assert L.tkv_evict_select_enqueue(C.byref(select(device=1 << 20, new_lens=A + 4096, **change)), None) == N.ERR_CUDA


@pytest.mark.parametrize("scale", [3e38, -3e38])
def test_attention_refuses_a_scale_that_is_infinite_in_the_log2_domain(L, scale):
    assert L.tkv_scored_attn_enqueue(C.byref(pool()), C.byref(scored(sm_scale=scale)), None) == BAD
    assert L.tkv_prefix_attn_enqueue(C.byref(pool()), C.byref(prefix(sm_scale=scale)), None) == BAD


@pytest.mark.parametrize("n_seqs,n_q_heads,n_kv_heads,head_dim,max_kv_len", [(64, 32, 8, 128, 4096), (1, 64, 8, 128, 131071), (3, 8, 1, 64, 100), (16, 32, 16, 128, 1)])
def test_the_scored_workspace_holds_one_partial_result_per_part_and_sequence(L, n_seqs, n_q_heads, n_kv_heads, head_dim, max_kv_len):
    """Scores of whole blocks, and (m, l, O) of at most 148 x 8 / min(kv heads, 8) parts and n_seqs sequences; the rest is a few words and alignment."""
    parts = 148 * 8 // min(n_kv_heads, 8) // -(-n_kv_heads // 8)
    scores = n_seqs * n_q_heads * -(-max_kv_len // 16) * 16 * 4
    got = L.tkv_scored_attn_scratch_bytes(n_seqs, n_q_heads, n_kv_heads, head_dim, max_kv_len)
    assert scores + n_seqs * n_q_heads * (head_dim + 2) * 4 < got <= scores + (parts + n_seqs) * n_q_heads * (head_dim + 2) * 4 + 4 * (n_seqs + 2) + 3 * 256
