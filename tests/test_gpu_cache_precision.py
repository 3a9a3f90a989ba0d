"""How exact the attention operators of the cache are, judged against the size of what is summed rather than against the largest V.

V is made so that a row's weighted sum nearly cancels: the rounding of the output to F16, 2^-11 of it, is then small, and what is left is the error
of the weights.  With w in 64 bits, A the largest sum of |scale log2(e) q_i k_i| of a row and n its tokens, an element of out may be off by
    2^-11 |out| + 2^-25 + sum_t w_t |v_t| * c,   c = 2 ln 2 A (D / 16 + 6) 2^-23 + (n / 8 + 24) 2^-23 + 2^-21:
a score is D / 16 truncating MMA steps and at most six roundings of terms whose sum of magnitudes is A (twice: in the weight and in the sum that it
is divided by); a row of O is two MMA steps per 16 tokens and at most 24 roundings (rescaling, joining, the sum's own); a probability of
22 bits and exp2 are 2^-23 and 2^-22 each, at both places.  A probability of one F16 term is off by up to 2^-11: the tests plant that in a plain
implementation and require that the bound catches it."""
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


def cancel(w, v, to):
    """Row `to` of v so that w @ v is about zero (w: one row of weights)."""
    rest = w @ v - w[to] * v[to]
    v[to] = -rest / w[to]


def bound(w, v, a, dim):
    """Per element of w @ v, see above."""
    n = v.shape[0]
    c = 2 * math.log(2) * a * (dim / 16 + 6) * 2.0 ** -23 + (n / 8 + 24) * 2.0 ** -23 + 2.0 ** -21
    return 2.0 ** -11 * (w @ v).abs() + 2.0 ** -25 + c * (w @ v.abs())


def one_term(q, k, v, scale):
    """The same attention with every probability rounded to F16 once, relative to its row's largest."""
    import torch
    x = q @ k.T * scale
    p = torch.exp(x - x.amax(dim=1, keepdim=True))
    return p.to(torch.float16).double() @ v / p.sum(dim=1, keepdim=True)


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


def cancelling_rows(q, n, kv_heads, dim, g, dtype, scale):
    """K and V [n, kv_heads, dim] for which a query row q [dim] attends to a sum of about zero."""
    import torch
    k = torch.randn((n, kv_heads, dim), generator=g, dtype=torch.float64)
    v = torch.randn((n, kv_heads, dim), generator=g, dtype=torch.float64)
    k, v = k.to(torch.float16).double(), v.to(torch.float16).double()
    for h in range(kv_heads):
        w, _ = weights(q[None], k[:, h], scale)
        cancel(w[0], v[:, h], int(w[0].argmax()))
    return k, v


def judge(out, q, case, s, h, group, scale, planted=None):
    """Checks query heads of kv head h of sequence s; `planted` collects how far a one-term form is outside of the bound."""
    k, v = case.k[s][:, h], case.v[s][:, h]
    rows = slice(h * group, (h + 1) * group)
    w, a = weights(q[s][rows].double(), k, scale)
    b = bound(w, v, a, case.dim)
    err = (out[s][rows].double().cpu() - w @ v).abs()
    assert (err <= b).all(), f"sequence {s}, kv head {h}: off by {(err / b).max():.2f} of the bound"
    if planted is not None:
        planted.append(float(((one_term(q[s][rows].double(), k, v, scale) - w @ v).abs() / b).max()))


@pytest.mark.parametrize("dtype", ["f16", "e4m3", "e4m3 unscaled"])
@pytest.mark.parametrize("kv_heads,dim,group", [(2, 128, 4), (3, 64, 8), (1, 128, 2)])
def test_scored_attention_keeps_both_terms_of_a_probability(H, dtype, kv_heads, dim, group):
    import torch
    g = torch.Generator().manual_seed(dim + group)
    lens, scale = [2, 3, 7, 16, 20, 40], 1 / math.sqrt(dim)
    q1 = torch.randn((len(lens), dim), generator=g).to(torch.float16)
    rows = [cancelling_rows(q1[s].double(), n, kv_heads, dim, g, dtype, scale) for s, n in enumerate(lens)]
    case = Case(H, dtype, kv_heads, dim, rows)
    q = q1[:, None].repeat(1, kv_heads * group, 1)
    scores = torch.zeros((1, len(lens), kv_heads, 48)).cuda()
    attn = H.ScoredDecodeAttention(case.pool, q.cuda(), case.tables.cuda(), torch.tensor(lens, dtype=torch.int32).cuda(), scores, 48)
    out, planted = attn.enqueue(0), []
    assert int(attn.status.item()) == 0
    for s in range(len(lens)):
        for h in range(kv_heads):
            judge(out, q, case, s, h, group, scale, planted)
    assert max(planted) > 2                                           # what is tested for would show


@pytest.mark.parametrize("dtype", ["f16", "e4m3", "e4m3 unscaled"])
@pytest.mark.parametrize("kv_heads,dim,group,members", [(2, 128, 4, 3), (3, 64, 8, 20), (1, 128, 2, 140)])
def test_prefix_attention_keeps_both_terms_of_a_probability(H, dtype, kv_heads, dim, group, members):
    """Groups that are nothing but their prefix: one tile, a short tile, and several steps."""
    import torch
    g = torch.Generator().manual_seed(dim + group + members)
    prefixes, scale = [16, 48, 64], 1 / math.sqrt(dim)
    q1 = torch.randn((len(prefixes), dim), generator=g).to(torch.float16)
    rows = [cancelling_rows(q1[i].double(), n, kv_heads, dim, g, dtype, scale) for i, n in enumerate(prefixes)]
    case = Case(H, dtype, kv_heads, dim, rows)
    of = torch.arange(len(prefixes)).repeat_interleave(members)
    case.k, case.v = [case.k[i] for i in of], [case.v[i] for i in of]
    q = q1[of][:, None].repeat(1, kv_heads * group, 1)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32).cuda()  # noqa: E731
    attn = H.PrefixAttention(case.pool, q.cuda(), case.tables[of].contiguous().cuda(), i32([prefixes[i] for i in of]),
                             i32([members * i for i in range(len(prefixes) + 1)]), i32(prefixes), max(prefixes), max(prefixes))
    out, planted = attn.enqueue(0), []
    assert int(attn.status.item()) == 0
    for s in range(0, len(of), max(1, members // 3)):
        for h in range(kv_heads):
            judge(out, q, case, s, h, group, scale, planted)
    assert max(planted) > 2


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
