"""Select at the row lengths where its work is split differently: one CTA, staged clusters of two, four and eight, a cluster whose slices do not fit
shared memory; several rows per launch, short and uncut rows inside a clustered launch."""

import ctypes

import numpy as np
import pytest

from tempura_b200 import _native as N

from test_gpu_cache_eviction import H, check_choice  # noqa: F401  (H is the fixture)

pytestmark = pytest.mark.gpu


def tied(shape, seed):
    """Scores of which half are zero and the first row of kv heads has only 101 values: ties reach across CTAs."""
    scores = np.random.default_rng(seed).random(shape, dtype=np.float32)
    scores[scores < 0.5] = 0.0
    scores[:, :, 0] = np.round(scores[:, :, 0], 2)
    return scores


@pytest.mark.parametrize("shape,lens", [
    ((2, 3, 2, 40000), [40000, 17, 33000]),                           # two CTAs a row; the second sequence ends inside what is kept
    ((1, 4, 1, 32769), [32769, 32768, 0, 1]),                         # the shortest rows that are split
    ((2, 2, 1, 100000), [65, 100000]),                                # four
    ((1, 2, 1, 300000), [300000, 140001]),                            # eight, the slices in shared memory
    ((1, 3, 1, 400001), [400001, 7, 400000]),                         # eight, too long for it
])
def test_rows_that_a_cluster_shares(H, shape, lens):  # noqa: F811
    scores = tied(shape, shape[3])
    for budget in (100, shape[3] // 3, shape[3] - 5):
        check_choice(H, scores, lens, [0] * len(lens), budget, 64)
    check_choice(H, scores, lens, [min(t, 33) for t in lens], 500, 10)


@pytest.mark.parametrize("shape,lens", [((3, 1, 4, 9000), [8999]), ((1, 2, 2, 30000), [30000, 17]), ((1, 2, 1, 32768), [32768, 20000]), ((2, 5, 80, 1100), [1100, 3, 1025, 0, 700])])
def test_rows_of_one_cta(H, shape, lens):  # noqa: F811
    scores = tied(shape, shape[3])
    for budget in (100, shape[3] // 3, shape[3] - 5):
        check_choice(H, scores, lens, [0] * len(lens), budget, 64)


@pytest.mark.parametrize("bound", [0xFFFFFFFF, 0xFFFFFFF9, 0xFFFFFFF8, 1 << 31])
def test_a_length_bound_at_the_end_of_32_bits(H, bound):  # noqa: F811
    """One row whose length is far below a bound that no row could reach: the bound decides how a row is split, and must not wrap."""
    import torch
    scores = torch.rand(500, generator=torch.Generator().manual_seed(1)).cuda()
    lens, kept, new, status = (torch.zeros(n, dtype=torch.int32).cuda() for n in (1, 64, 1, 1))
    lens.fill_(500)
    args = N.TkvEvictSelect(0, 1, 1, 1, bound, bound, 64, 64, 8, 0, scores.data_ptr(), lens.data_ptr(), 0, kept.data_ptr(), new.data_ptr(), status.data_ptr())
    torch.cuda.synchronize()
    assert N.lib().tkv_evict_select_enqueue(ctypes.byref(args), None) == 0
    torch.cuda.synchronize()
    top = sorted(torch.topk(scores[:492], 56).indices.tolist()) + list(range(492, 500))
    assert int(status) == 0 and int(new) == 64 and kept.tolist() == top
