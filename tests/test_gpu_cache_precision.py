"""How exact the attention operators of the cache are, judged against the size of what is summed rather than against the largest V.

With w in 64 bits, A the largest sum of |scale log2(e) q_i k_i| of a row and n its tokens, an element of out may be off by
    2^-11 |out| + 2^-25 + sum_t w_t |v_t| * c,   c = 2 ln 2 A (D / 16 + 6) 2^-23 + (n / 8 + 24) 2^-23 + 2^-21:
a score is D / 16 truncating MMA steps and at most six roundings of terms whose sum of magnitudes is A (twice: in the weight and in the sum that it
is divided by); a row of O is two MMA steps per 16 tokens and at most 24 roundings (rescaling, joining, the sum's own); a probability of
22 bits and exp2 are 2^-23 and 2^-22 each, at both places."""
import math

import pytest

pytestmark = pytest.mark.gpu
BS = 16
LOG2E = 1.4426950408889634


@pytest.fixture(scope="module")
def H():
    import torch
    assert torch.cuda.is_available()
    from tempura_b200 import handoff
    return handoff


def e4m3(x):
    import torch
    return torch.where(x.abs() < 2.0 ** -6, torch.zeros_like(x), x).clamp(-448, 448).to(torch.float8_e4m3fn)


def weights(q, k, scale):
    """q [heads, D], k [n, D] in 64 bits: weights [heads, n], and the largest sum of |scale log2(e) q_i k_i|."""
    import torch
    return torch.softmax(q @ k.T * scale, dim=1), float((q.abs() @ k.abs().T).max()) * abs(scale) * LOG2E


def bound(w, v, a, dim):
    """Per element of w @ v, see above."""
    n = v.shape[0]
    c = 2 * math.log(2) * a * (dim / 16 + 6) * 2.0 ** -23 + (n / 8 + 24) * 2.0 ** -23 + 2.0 ** -21
    return 2.0 ** -11 * (w @ v).abs() + 2.0 ** -25 + c * (w @ v.abs())


class Case:
    """One pool whose sequences (or prefix) hold given K and V rows [tokens, kv_heads, D]; E4M3 pools with given V block scales."""

    def __init__(self, H, dtype, kv_heads, dim, rows, v_scale=None, seed=0):
        import torch
        self.kv_heads, self.dim = kv_heads, dim
        counts = [(k.shape[0] + BS - 1) // BS for k, _ in rows]
        total = sum(counts) + 2
        perm = torch.randperm(total, generator=torch.Generator().manual_seed(seed))
        self.pool = H.Pool.allocate(0, 1, kv_heads, dim, BS, total, "f16" if dtype == "f16" else "e4m3", scales=dtype == "e4m3", fill_byte=None)
        self.tables = torch.full((len(rows), max(counts)), -1, dtype=torch.int32)
        self.k, self.v, at = [], [], 0
        for s, (k, v) in enumerate(rows):
            kept = [[], []]
            for b in range(counts[s]):
                block = int(perm[at])
                at += 1
                self.tables[s, b] = block
                for is_v, x in ((False, k), (True, v)):
                    x = x[b * BS: (b + 1) * BS]
                    view = self.pool.blocks(0, is_v)[block, : x.shape[0]]
                    if dtype == "f16":
                        y = x.to(torch.float16)
                        view.copy_(y)
                        kept[is_v].append(y.double())
                        continue
                    sc = (x.abs().amax(dim=(0, 2)) / 448).clamp_min(1e-9).float() if dtype == "e4m3" else torch.ones(kv_heads)
                    y = e4m3((x / sc[None, :, None]).float())
                    view.copy_(y.view(torch.uint8))
                    kept[is_v].append(y.float().double() * sc.double()[None, :, None])
                    if dtype == "e4m3":
                        (self.pool.v_scales if is_v else self.pool.k_scales)[0, block].copy_(sc)
            self.k.append(torch.cat(kept[0]))
            self.v.append(torch.cat(kept[1]))


def judge(out, q, case, s, h, group, scale):
    """Checks query heads of kv head h of sequence s."""
    k, v = case.k[s][:, h], case.v[s][:, h]
    rows = slice(h * group, (h + 1) * group)
    w, a = weights(q[s][rows].double(), k, scale)
    b = bound(w, v, a, case.dim)
    err = (out[s][rows].double().cpu() - w @ v).abs()
    assert (err <= b).all(), f"sequence {s}, kv head {h}: off by {(err / b).max():.2f} of the bound"


def spread_rows(n, loud, ratio, dim, g, q):
    """One kv head, n tokens; V of block `loud` is `ratio` times larger, and query q finds next to nothing there: some 2^-40."""
    import torch
    k = torch.randn((n, 1, dim), generator=g, dtype=torch.float64) * 0.5
    v = torch.randn((n, 1, dim), generator=g, dtype=torch.float64)
    v[loud * BS: (loud + 1) * BS] *= ratio
    k[loud * BS: (loud + 1) * BS] = -q * 28 * math.sqrt(dim) / float(q @ q)
    return k, v


@pytest.mark.parametrize("ratio", [2.0 ** 10, 2.0 ** 16, 2.0 ** 24])
@pytest.mark.parametrize("loud", [0, 1, 4])
def test_a_block_with_a_large_scale_and_no_weight_costs_the_others_nothing(H, ratio, loud):
    """Scaled E4M3 pool: the error stays small against the output, whatever the scales of blocks that do not count.  The opposite query puts all
    weight on that block."""
    import torch
    dim, group, n = 128, 4, 75
    g = torch.Generator().manual_seed(loud)
    scale = 1 / math.sqrt(dim)
    q1 = torch.randn(dim, generator=g).to(torch.float16)
    case = Case(H, "e4m3", 1, dim, [spread_rows(n, loud, ratio, dim, g, q1.double())])
    case.k, case.v, tables = case.k * 4, case.v * 4, case.tables.repeat(4, 1).contiguous()
    sign = torch.tensor([1.0, -1.0, 1.0, -1.0], dtype=torch.float16)
    q = (q1[None, None] * sign[:, None, None]).repeat(1, group, 1)
    q[:, 1::2] *= 0.5
    lens = torch.full((4,), n, dtype=torch.int32).cuda()
    scored = H.ScoredDecodeAttention(case.pool, q.cuda(), tables.cuda(), lens, torch.zeros((1, 4, 1, 80)).cuda(), n)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32).cuda()  # noqa: E731
    pre = H.PrefixAttention(case.pool, q.cuda(), tables.cuda(), lens, i32([0, 4]), i32([64]), n, 64)
    for attn in (scored, pre):
        out = attn.enqueue(0)
        assert int(attn.status.item()) == 0
        for s in range(4):
            if s % 2 and ratio > 2.0 ** 10:                           # the sum itself is past F16's range there
                continue
            judge(out, q, case, s, 0, group, scale)
