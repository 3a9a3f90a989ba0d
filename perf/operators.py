"""Measured cases of the operators that work on a paged KV cache while a batch decodes: attention of sequences that share a
prefix, attention that also accumulates how much weight every cached token got, the choice of the tokens that stay when a cache
is cut to a budget, and the move of their rows inside the cache.

``run`` computes an operator in elementary torch operations, or calls the framework where ``own`` is true.  ``exact`` computes
the same outputs from the definitions in 64 bits.  Shapes are those of the benchmark's models (kv heads x head_dim x query heads
per kv head: 4 x 64 x 8, 8 x 128 x 4, 8 x 128 x 8 and its shards over 2, 4 and 8 GPUs) and a few generic ones.
"""
import math
import random

import torch

own = False

BLOCK = 16                                  # tokens of a pool block
GEOMETRIES = [(4, 64, 8), (8, 128, 4), (8, 128, 8), (4, 128, 8), (2, 128, 8), (1, 128, 8), (1, 128, 4), (2, 64, 8), (6, 64, 1), (5, 128, 3)]
MOST_PREFIX = 128 * 16640 * 8 * 128         # (sequence, token, kv head, dim) cells of the largest listed case of each operator
MOST_PREFIX_FLOPS = 4 * 128 * 64 * 16640 * 128
MOST_SCORED = 64 * 4096 * 8 * 128
MOST_SELECT = 32 * 16 * 8 * 4096
MOST_COMPACT = 16 * 16 * 4096 * 8 * 128


def _geometry(kv_heads, head_dim, group):
    return {"kv_heads": kv_heads, "head_dim": head_dim, "group": group}


def listed():
    tiny, mid, large = _geometry(4, 64, 8), _geometry(8, 128, 4), _geometry(8, 128, 8)
    return [
        # three chats over one short system prompt: nothing but launch and memory latency
        {"name": "prefix 3 x 48", "op": "prefix", "pool": "f16", **tiny, "seqs": 3, "groups": 1, "prefix_lo": 48, "prefix_hi": 48, "suffix_lo": 1,
         "suffix_hi": 20, "lens": 1},
        # the benchmark's prefix batch: 64 prompts on one 2 048-token prefix, 128 to 512 tokens of their own
        {"name": "prefix 64 x 2048", "op": "prefix", "pool": "f16", **mid, "seqs": 64, "groups": 1, "prefix_lo": 2048, "prefix_hi": 2048,
         "suffix_lo": 128, "suffix_hi": 512, "lens": 2},
        # an FP8 cache serving several prompts' families at once, uneven groups and lengths, some sequences with no token of their own yet
        {"name": "prefix e4m3 45 in 7", "op": "prefix", "pool": "e4m3", **mid, "seqs": 45, "groups": 7, "prefix_lo": 200, "prefix_hi": 9000,
         "suffix_lo": 0, "suffix_hi": 700, "lens": 3},
        # many answers about one long document, 64 query heads: bound by arithmetic, not by the cache
        {"name": "prefix 128 x 16384", "op": "prefix", "pool": "f16", **large, "seqs": 128, "groups": 1, "prefix_lo": 16384, "prefix_hi": 16384,
         "suffix_lo": 32, "suffix_hi": 256, "lens": 4},
        # one short chat whose cache is watched for eviction
        {"name": "scored 1 x 200", "op": "scored", "pool": "f16", **tiny, "seqs": 1, "len_lo": 200, "len_hi": 200, "decay": 1.0, "lens": 5},
        # the benchmark's 16 prompts of 512 to 4 096 tokens
        {"name": "scored 16 x 4096", "op": "scored", "pool": "f16", **mid, "seqs": 16, "len_lo": 512, "len_hi": 4096, "decay": 1.0, "lens": 6},
        # a full FP8 batch with forgetting
        {"name": "scored e4m3 64 x 4096", "op": "scored", "pool": "e4m3", **mid, "seqs": 64, "len_lo": 512, "len_hi": 4096, "decay": 0.98, "lens": 7},
        # one long context: the work has to be split over the tokens
        {"name": "scored 1 x 131071", "op": "scored", "pool": "f16", **large, "seqs": 1, "len_lo": 131071, "len_hi": 131071, "decay": 1.0, "lens": 8},
        # one short chat, all layers
        {"name": "select 22 x 512", "op": "select", **tiny, "layers": 22, "seqs": 1, "len_lo": 512, "len_hi": 512, "budget": 128, "recent": 32,
         "protect_hi": 4, "lens": 9},
        # the benchmark's 16 prompts cut to 1 024 tokens in all layers
        {"name": "select 32 x 16 x 4096", "op": "select", **mid, "layers": 32, "seqs": 16, "len_lo": 512, "len_hi": 4096, "budget": 1024,
         "recent": 128, "protect_hi": 64, "lens": 10},
        # the same prompts' rows moved, 16 layers
        {"name": "compact 16 x 16 x 4096", "op": "compact", "pool": "f16", **mid, "layers": 16, "seqs": 16, "len_lo": 512, "len_hi": 4096,
         "budget": 1024, "recent": 128, "protect_hi": 0, "lens": 11},
        # an FP8 cache with scales, shared prefixes protected, odd budget
        {"name": "compact e4m3 32 x 7", "op": "compact", "pool": "e4m3", **mid, "layers": 32, "seqs": 7, "len_lo": 300, "len_hi": 4096,
         "budget": 701, "recent": 100, "protect_hi": 256, "lens": 12},
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    op = rng.choice(["prefix", "scored", "select", "compact"])
    kv_heads, head_dim, group = rng.choice(GEOMETRIES)
    case = {"op": op, **_geometry(kv_heads, head_dim, group), "lens": rng.randrange(1 << 30)}
    if op != "select":
        case["pool"] = rng.choice(["f16", "e4m3", "e4m3 unscaled"])
    if op == "prefix":
        case["seqs"] = _log(rng, 1, 128)
        case["groups"] = rng.randint(1, min(8, case["seqs"]))
        hi = _log(rng, 16, 16384)
        case["suffix_hi"] = _log(rng, 1, 512)
        case["suffix_lo"] = rng.choice([0, 1, case["suffix_hi"] // 2])
        while case["seqs"] * (hi + case["suffix_hi"]) * kv_heads * head_dim > MOST_PREFIX or 4 * case["seqs"] * kv_heads * group * (hi + 512) * head_dim > MOST_PREFIX_FLOPS:
            hi //= 2
        case["prefix_hi"] = hi
        case["prefix_lo"] = rng.choice([0, hi // 3, hi])
    else:
        if op == "scored":
            case["seqs"] = _log(rng, 1, 64)
            hi, most, layers = _log(rng, 1, 131071), MOST_SCORED, 1
            case["decay"] = rng.choice([1.0, 0.9, 0.0])
        else:
            case["layers"] = layers = _log(rng, 1, 32 if op == "select" else 16)
            case["seqs"] = _log(rng, 1, 16)
            hi, most = _log(rng, 16, 65536 if op == "select" else 8192), MOST_SELECT if op == "select" else MOST_COMPACT
        cells = kv_heads * (1 if op == "select" else head_dim)
        while layers * case["seqs"] * hi * cells > most:
            hi = hi * 2 // 3
        hi = max(hi, 1)
        case["len_hi"] = hi
        case["len_lo"] = rng.choice([1, max(1, hi // 4), hi])
        if op != "scored":
            case["budget"] = _log(rng, 1, hi)
            case["recent"] = rng.choice([0, 1, case["budget"] // 4])
            case["protect_hi"] = rng.choice([0, 4, case["budget"] // 3])
    return case


# ---- what the case alone decides: lengths and groups --------------------------------------------------------------------------
def _plan(case):
    rng = random.Random(case["lens"])
    n = case["seqs"]
    if case["op"] == "prefix":
        cuts = sorted(rng.sample(range(1, n), case["groups"] - 1))
        starts = [0] + cuts + [n]
        prefix = [rng.randint(case["prefix_lo"], case["prefix_hi"]) // BLOCK * BLOCK for _ in range(case["groups"])]
        of = [g for g in range(case["groups"]) for _ in range(starts[g], starts[g + 1])]
        lens = [prefix[of[s]] + rng.randint(case["suffix_lo"], case["suffix_hi"]) for s in range(n)]
        lens[-1] = max(1, lens[-1])
        return {"starts": starts, "prefix": prefix, "of": of, "lens": lens}
    lens = [rng.randint(case["len_lo"], case["len_hi"]) for _ in range(n)]
    if case["op"] == "scored":
        return {"lens": lens}
    protect = [rng.randint(0, case["protect_hi"]) // (BLOCK if case["op"] == "compact" else 1) * (BLOCK if case["op"] == "compact" else 1) for _ in range(n)]
    new = [min(l, max(case["budget"], p + case["recent"])) for l, p in zip(lens, protect)]
    return {"lens": lens, "protect": protect, "new": new}


def work(case):
    p, h, d, g, n = _plan(case), case["kv_heads"], case["head_dim"], case["group"], case["seqs"]
    es = 2 if case.get("pool") == "f16" else 1
    scales = 1 if case.get("pool") == "e4m3" else 0
    blocks = lambda t: -(-t // BLOCK)  # noqa: E731
    per_token = 2 * h * d * es
    per_block = 2 * h * 4 * scales + 4                      # scales of K and V, the table entry
    q_out = 2 * n * h * g * d * 2
    if case["op"] == "prefix":
        own_tokens = [l - p["prefix"][p["of"][s]] for s, l in enumerate(p["lens"])]
        tokens = sum(p["prefix"]) + sum(own_tokens)
        n_blocks = sum(blocks(t) for t in p["prefix"]) + sum(blocks(t) for t in own_tokens)
        return {"bytes": tokens * per_token + n_blocks * per_block + q_out, "flops": 4 * h * g * d * sum(p["lens"])}
    if case["op"] == "scored":
        tokens = sum(p["lens"])
        score = 4 * h * tokens * (2 if case["decay"] else 1)
        return {"bytes": tokens * per_token + sum(blocks(t) for t in p["lens"]) * per_block + q_out + score, "flops": 4 * h * g * d * tokens}
    rows = case["layers"] * h
    if case["op"] == "select":
        return {"bytes": rows * (sum(p["lens"]) + sum(p["new"])) * 4, "flops": rows * sum(p["lens"])}
    moved = sum(max(0, m - q) for l, q, m in zip(p["lens"], p["protect"], p["new"]) if m < l)
    cut = sum(l - m for l, m in zip(p["lens"], p["new"]))
    return {"bytes": rows * (2 * moved * (2 * d * es + 4) + 4 * sum(p["new"]) + 4 * cut), "flops": rows * moved * d * (2 if scales else 0)}


# ---- inputs -----------------------------------------------------------------------------------------------------------------
def _pool(gen, layers, n_blocks, case):
    """K or V of all layers: normal values with one channel of outliers, as block values (and scales) of the pool's type."""
    h, d = case["kv_heads"], case["head_dim"]
    x = torch.empty((layers, n_blocks, BLOCK, h, d), dtype=torch.float16, device="cuda").normal_(0.0, 0.5, generator=gen)
    x[..., d // 3] *= 6.0
    if case["pool"] == "f16":
        return x, None
    data = torch.empty(x.shape, dtype=torch.float8_e4m3fn, device="cuda")
    scale = None
    if case["pool"] == "e4m3":
        scale = (x.abs().amax(dim=(2, 4)).float() / 448.0).clamp_min(1e-8)
    for layer in range(layers):
        y = x[layer].float()
        if scale is not None:
            y = (y / scale[layer][:, None, :, None]).clamp(-448.0, 448.0)
        data[layer] = torch.where(y.abs() < 2.0 ** -6, torch.zeros_like(y), y).to(torch.float8_e4m3fn)
    return data, scale


def _tables(gen, lens, prefix=None, of=None):
    """Block tables over a shuffled pool: the members of a group name the same blocks for their prefix."""
    n, width = len(lens), max(1, max(-(-t // BLOCK) for t in lens))
    count, rows, shared = 0, [], {}
    for s, t in enumerate(lens):
        need, row = -(-t // BLOCK), []
        if prefix is not None:
            g = of[s]
            if g not in shared:
                shared[g] = list(range(count, count + prefix[g] // BLOCK))
                count += len(shared[g])
            row = list(shared[g])
        row += list(range(count, count + need - len(row)))
        count = max(count, row[-1] + 1 if row else 0)
        rows.append(row + [0] * (width - need))
    total = count + 5
    perm = torch.randperm(total, generator=gen, device="cuda")
    return perm[torch.tensor(rows, device="cuda")].to(torch.int32), total


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    p, n, h, d, g = _plan(case), case["seqs"], case["kv_heads"], case["head_dim"], case["group"]
    dev = "cuda"
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)  # noqa: E731
    st = {"case": case, "plan": p, "lens": i32(p["lens"]), "max_len": max(p["lens"])}
    if case["op"] in ("prefix", "scored"):
        st["tables"], total = _tables(gen, p["lens"], p.get("prefix"), p.get("of"))
        st["k"], st["k_scales"] = _pool(gen, 1, total, case)
        st["v"], st["v_scales"] = _pool(gen, 1, total, case)
        st["q"] = torch.empty((n, h * g, d), dtype=torch.float16, device=dev).normal_(0.0, 2.0, generator=gen)
        st["sm_scale"] = 1.0 / math.sqrt(d)
    if case["op"] == "prefix":
        st["starts"], st["prefix"] = i32(p["starts"]), i32(p["prefix"])
    elif case["op"] == "scored":
        # what a few earlier steps left, in the order of one step's weights
        st["scores"] = torch.rand((1, n, h, st["max_len"]), generator=gen, device=dev) * (4.0 / st["lens"].clamp_min(1).float())[None, :, None, None]
    else:
        layers = case["layers"]
        st["protect"] = i32(p["protect"])
        # accumulated weights: most tokens little, a few much; a share of them never looked at (equal scores)
        s = torch.empty((layers, n, h, st["max_len"]), device=dev).exponential_(1.0, generator=gen) ** 3
        st["scores"] = torch.where(torch.rand(s.shape, generator=gen, device=dev) < 0.1, torch.zeros_like(s), s)
        width = max(p["new"])
        st["kept"] = torch.zeros((layers, n, h, width), dtype=torch.int32, device=dev)
        st["new"] = torch.zeros(n, dtype=torch.int32, device=dev)
        if case["op"] == "compact":
            st["kept"], st["new"] = _choose(st["scores"], st["lens"], st["protect"], case["budget"], case["recent"], width)
            st["tables"], total = _tables(gen, p["lens"])
            st["k"], st["k_scales"] = _pool(gen, layers, total, case)
            st["v"], st["v_scales"] = _pool(gen, layers, total, case)
    return st


# ---- plain forms ------------------------------------------------------------------------------------------------------------
def _gathered(data, scales, tables, length):
    """f32 [sequence, token, kv head, dim] of one layer, and which tokens exist."""
    x = data[tables.long()].float()
    if scales is not None:
        x = x * scales[tables.long()][:, :, None, :, None]
    return x.flatten(1, 2)[:, :length]


def _attention(st, length):
    q, lens = st["q"].float(), st["lens"]
    n, hq, d = q.shape
    k = _gathered(st["k"][0], None if st["k_scales"] is None else st["k_scales"][0], st["tables"], length)
    h = k.shape[2]
    s = torch.matmul(q.view(n, h, hq // h, d), k.permute(0, 2, 3, 1)) * st["sm_scale"]
    del k
    live = (torch.arange(length, device=q.device)[None, :] < lens[:, None])[:, None, None, :]
    s = torch.where(live, s, torch.full_like(s, -math.inf))
    m = s.amax(dim=-1, keepdim=True)
    w = torch.where(live, torch.exp(s - m), torch.zeros_like(s))
    total = w.sum(dim=-1, keepdim=True)
    w = torch.where(total > 0, w / total, torch.zeros_like(w))
    v = _gathered(st["v"][0], None if st["v_scales"] is None else st["v_scales"][0], st["tables"], length)
    out = torch.matmul(w, v.permute(0, 2, 1, 3)).view(n, hq, d)
    return out.to(st["q"].dtype), w


def _choose(scores, lens, protect, budget, recent, width):
    """Indices kept, ascending; ties to the lower index; protected heads and recent tails always stay."""
    length = scores.shape[-1]
    t = torch.arange(length, device=scores.device)
    lens, protect = lens.long(), protect.long()
    new = torch.minimum(lens, torch.clamp_min(protect + recent, budget))
    always = ((t[None] < protect[:, None]) | (t[None] >= (lens - recent)[:, None]))[None, :, None, :]
    exists = (t[None] < lens[:, None])[None, :, None, :]
    key = torch.where(always, torch.full_like(scores, math.inf), scores)
    key = torch.where(exists, key, torch.full_like(scores, -math.inf))
    order = torch.sort(key, dim=-1, descending=True, stable=True).indices[..., :width]
    taken = (torch.arange(width, device=scores.device)[None] < new[:, None])[None, :, None, :]
    order = torch.sort(torch.where(taken, order, torch.full_like(order, length)), dim=-1).values
    return torch.where(taken, order, torch.zeros_like(order)).to(torch.int32), new.to(torch.int32)


def _moved(data, scales, src, dst, layer, head, live):
    """Rows of one tensor in their new places, and the scales of the blocks they now are in."""
    rows = data.flatten(1, 2)
    picked = rows.view(torch.uint8 if rows.dtype != torch.float16 else torch.float16)[layer, src, head]
    if scales is not None:
        old = scales[layer, src // BLOCK, head]
        pad = -old.shape[-1] % BLOCK
        padded = torch.nn.functional.pad(torch.where(live, old, torch.full_like(old, -math.inf)), (0, pad), value=-math.inf)
        new = padded.unflatten(-1, (-1, BLOCK)).amax(dim=-1)
        ratio = (old / new.repeat_interleave(BLOCK, dim=-1)[..., : old.shape[-1]])[..., None]
        x = picked.view(torch.float8_e4m3fn).float() * ratio
        x = torch.where(x.abs() < 2.0 ** -6, x * 0.0, x).to(torch.float8_e4m3fn).view(torch.uint8)
        picked = torch.where(ratio == 1.0, picked, x)
        first = (layer.expand_as(dst)[..., ::BLOCK], (dst // BLOCK)[..., ::BLOCK], head.expand_as(dst)[..., ::BLOCK])
        scales[first] = torch.where(live[..., ::BLOCK], new, scales[first])
    flat = rows.view(picked.dtype)
    flat[layer, dst, head] = torch.where(live[..., None], picked, flat[layer, dst, head])


def run(state):
    case = state["case"]
    if own:
        return _own(state)
    if case["op"] == "prefix":
        return _attention(state, state["max_len"])[0]
    if case["op"] == "scored":
        out, w = _attention(state, state["max_len"])
        w = w.sum(dim=2)                    # over the query heads of a kv head
        live = (torch.arange(w.shape[-1], device=w.device)[None, :] < state["lens"][:, None])[:, None, :]
        kept = state["scores"][0] * case["decay"] if case["decay"] else torch.zeros_like(w)
        state["scores"][0] = torch.where(live, kept + w, state["scores"][0])
        return {"out": out, "scores": state["scores"]}
    if case["op"] == "select":
        kept, new = _choose(state["scores"], state["lens"], state["protect"], case["budget"], case["recent"], state["kept"].shape[-1])
        return {"kept": kept, "new": new}
    kept, new, tables = state["kept"].long(), state["new"].long(), state["tables"].long()
    layers, n, h, width = kept.shape
    j = torch.arange(width, device=kept.device)
    live = (j[None] < new[:, None])[None, :, None, :].expand_as(kept)
    src_token = torch.where(live, kept, torch.zeros_like(kept))
    seq = torch.arange(n, device=kept.device)[None, :, None, None]
    src = tables[seq, src_token // BLOCK] * BLOCK + src_token % BLOCK
    # slots past the new length write nothing: they go to the row of the pool that no table names
    used = torch.zeros(state["k"].shape[1], dtype=torch.int32, device=kept.device)
    used[tables.flatten()] = 1
    free = torch.argmin(used)
    dst = torch.where(live, tables[seq, (j // BLOCK)[None, None, None, :]] * BLOCK + j % BLOCK, free * BLOCK + j % BLOCK)
    layer = torch.arange(layers, device=kept.device)[:, None, None, None]
    head = torch.arange(h, device=kept.device)[None, None, :, None]
    _moved(state["k"], state["k_scales"], src, dst, layer, head, live)
    _moved(state["v"], state["v_scales"], src, dst, layer, head, live)
    scores = state["scores"]
    t = torch.arange(scores.shape[-1], device=kept.device)
    picked = torch.gather(scores, -1, src_token)
    exists = (t[None] < state["lens"][:, None])[None, :, None, :]
    stays = torch.nn.functional.pad(torch.where(live, picked, torch.zeros_like(picked)), (0, scores.shape[-1] - width))
    scores.copy_(torch.where(exists, stays, scores))
    return {k: state[k] for k in ("k", "v", "k_scales", "v_scales", "scores") if state[k] is not None}


# ---- the framework's calls --------------------------------------------------------------------------------------------------
def _handle(state):
    from tempura_b200 import handoff as H
    case = state["case"]
    if case["op"] == "select":
        return H.CacheEviction(None, None, state["lens"], state["scores"], case["budget"], case["recent"], protect=state["protect"],
                               kept=state["kept"], new_lens=state["new"])
    k, v = state["k"], state["v"]
    pointers = lambda x: [x[layer].data_ptr() for layer in range(x.shape[0])]  # noqa: E731
    ks, vs = ((x.data_ptr() if x is not None else 0) for x in (state["k_scales"], state["v_scales"]))
    pool = H.Pool.from_pointers(0, "f16" if case["pool"] == "f16" else "e4m3", case["kv_heads"], case["head_dim"], BLOCK, k.shape[1],
                                pointers(k), pointers(v), ks, vs)
    if case["op"] == "prefix":
        return H.PrefixAttention(pool, state["q"], state["tables"], state["lens"], state["starts"], state["prefix"], state["max_len"],
                                 max(state["plan"]["prefix"]), sm_scale=state["sm_scale"])
    if case["op"] == "scored":
        return H.ScoredDecodeAttention(pool, state["q"], state["tables"], state["lens"], state["scores"], state["max_len"],
                                       sm_scale=state["sm_scale"], decay=case["decay"])
    return H.CacheEviction(pool, state["tables"], state["lens"], state["scores"], case["budget"], case["recent"], protect=state["protect"],
                           kept=state["kept"], new_lens=state["new"])


def _own(state):
    op = state["case"]["op"]
    if "handle" not in state:               # made once and kept, with its workspace, as a decode loop does
        state["handle"] = _handle(state)
    handle = state["handle"]
    if op == "prefix":
        return handle.enqueue(0)
    if op == "scored":
        return {"out": handle.enqueue(0), "scores": state["scores"]}
    if op == "select":
        handle.select()
        return {"kept": state["kept"], "new": state["new"]}
    handle.compact()
    return {k: state[k] for k in ("k", "v", "k_scales", "v_scales", "scores") if state[k] is not None}


# ---- 64 bits ----------------------------------------------------------------------------------------------------------------
def _rows64(st, name, layer, seq, tokens, head):
    """Values of some tokens of one sequence and kv head."""
    block = st["tables"][seq].long()[tokens // BLOCK]
    x = st[name][layer, block, tokens % BLOCK, head]
    x = x.double() if x.dtype == torch.float16 else x.float().double()
    if st[name + "_scales"] is not None:
        x = x * st[name + "_scales"][layer, block, head].double()[:, None]
    return x


def exact(case, seed):
    st = prepare(case, seed)
    p, n, h, g = st["plan"], case["seqs"], case["kv_heads"], case["group"]
    if case["op"] in ("prefix", "scored"):
        if n * h > 2048:
            return None
        out = torch.zeros(st["q"].shape, dtype=torch.float64, device="cuda")
        scores = st["scores"].double() if case["op"] == "scored" else None
        for s in range(n):
            t = torch.arange(p["lens"][s], device="cuda")
            for head in range(h):
                if not len(t):
                    continue
                q = st["q"][s, head * g: (head + 1) * g].double()
                x = q @ _rows64(st, "k", 0, s, t, head).T * st["sm_scale"]
                x = torch.exp(x - x.max(dim=1, keepdim=True).values)
                x = x / x.sum(dim=1, keepdim=True)
                out[s, head * g: (head + 1) * g] = x @ _rows64(st, "v", 0, s, t, head)
                if scores is not None:
                    scores[0, s, head, : len(t)] = case["decay"] * scores[0, s, head, : len(t)] + x.sum(dim=0)
        return out if scores is None else {"out": out, "scores": scores}
    if case["op"] == "select":
        return None                         # whole numbers
    if case["layers"] * n * h > 5000:
        return None
    fresh = {}
    for name in ("k", "v"):
        old, scales = st[name], st[name + "_scales"]
        x = (old if old.dtype == torch.float16 else old.float()).double()
        new_scales = None if scales is None else scales.double()
        for layer in range(case["layers"]):
            for s in range(n):
                m = p["new"][s]
                j = torch.arange(m, device="cuda")
                to = st["tables"][s].long()[j // BLOCK]
                for head in range(h):
                    src = st["kept"][layer, s, head, :m].long()
                    at = st["tables"][s].long()[src // BLOCK]
                    row = old[layer, at, src % BLOCK, head]
                    row = (row if row.dtype == torch.float16 else row.float()).double()
                    if scales is not None:
                        sc = scales[layer, at, head].double()
                        top = torch.zeros(-(-m // BLOCK), dtype=torch.float64, device="cuda").scatter_reduce(0, j // BLOCK, sc, "amax")
                        new_scales[layer, to[::BLOCK], head] = top
                        row = row * (sc / top[j // BLOCK])[:, None]
                    x[layer, to, j % BLOCK, head] = row
        fresh[name] = x
        if scales is not None:
            fresh[name + "_scales"] = new_scales
    scores = st["scores"].double()
    for s in range(n):
        m, l = p["new"][s], p["lens"][s]
        moved = torch.gather(st["scores"][:, s].double(), -1, st["kept"][:, s, :, :m].long())
        scores[:, s, :, :l] = 0.0
        scores[:, s, :, :m] = moved
    fresh["scores"] = scores
    return fresh
