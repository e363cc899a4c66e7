"""The operators of a speculative decoding step, as cases that can be timed: a step in which every sequence brings a tree
of drafted tokens.

  step     the step's tables from request lengths, on the GPU: blocks taken from the free list, block tables, slots,
           positions, for a tree also its ancestor masks; and the blocks given back when the step is rolled back
  attn     attention of the drafted tokens over the paged cache that already holds their keys and values
  accept   the walk through the tree along the tokens that the target model sampled at its nodes
  compact  the accepted nodes' cache rows moved to their places behind the context, all layers

Heads are (query heads, kv heads) of one GPU: Qwen3-0.6B and Qwen3-8B geometry at tensor parallelism 1, 2, 4, 8.  Lengths
are spread evenly over their range (so the work of a case is known); their order, trees, block ids and values come from
the seed.  Blocks of 256 tokens scattered at random, bf16, head_dim 128.
"""
from __future__ import annotations

import math

import torch

own = False

BLOCK = 256
D = 128
LAYERS = 28
VOCAB = 151936
HEADS = ((16, 8), (8, 4), (4, 2), (2, 1), (32, 8), (16, 4), (8, 2), (4, 1))
DEV = "cuda"


def listed():
    return [
        # a full decode batch of the engine: one new token each, block tables of 4096 tokens
        dict(name="step_decode_512", op="step", batch=512, cached_lo=100, cached_hi=4000, new_lo=1, new_hi=1, tree=False, cols=16),
        # ragged prompts up to the engine's limit of 16384 tokens in a prefill step, nothing cached
        dict(name="step_prefill_40", op="step", batch=40, cached_lo=0, cached_hi=0, new_lo=39, new_hi=780, tree=False, cols=16),
        # trees of up to 64 drafted tokens, tables of 40960 tokens
        dict(name="step_tree_96", op="step", batch=96, cached_lo=90, cached_hi=9000, new_lo=17, new_hi=64, tree=True, cols=160),
        # one chat with a small tree: the smallest call, where latency counts
        dict(name="attn_one", op="attn", batch=1, ctx_lo=1037, ctx_hi=1037, new_lo=9, new_hi=9, H=16, Hkv=8, tree=True),
        # a lightly loaded server, odd sizes
        dict(name="attn_chat", op="attn", batch=13, ctx_lo=203, ctx_hi=3001, new_lo=5, new_hi=33, H=32, Hkv=8, tree=True),
        # drafts without branches (no masks: each sees those before it) on a busy server
        dict(name="attn_chain_busy", op="attn", batch=256, ctx_lo=100, ctx_hi=2048, new_lo=4, new_hi=4, H=16, Hkv=8, tree=False),
        # few requests with long contexts, on one GPU of four
        dict(name="attn_long", op="attn", batch=4, ctx_lo=24000, ctx_hi=40960, new_lo=33, new_hi=64, H=8, Hkv=2, tree=True),
        # large trees in a large batch of the 8B geometry: products weigh as much as bytes
        dict(name="attn_busy_8b", op="attn", batch=128, ctx_lo=512, ctx_hi=4096, new_lo=64, new_hi=64, H=32, Hkv=8, tree=True),
        # the walk after a small step, and after the largest
        dict(name="accept_13", op="accept", batch=13, new_lo=5, new_hi=33),
        dict(name="accept_512", op="accept", batch=512, new_lo=33, new_hi=64),
        # all layers' accepted rows: a few chats, and a busy server (one GPU of four)
        dict(name="compact_5", op="compact", batch=5, ctx_lo=100, ctx_hi=900, new_lo=17, new_hi=33, Hkv=8, path=6),
        dict(name="compact_128", op="compact", batch=128, ctx_lo=100, ctx_hi=440, new_lo=33, new_hi=64, Hkv=2, path=8),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    op = rng.choice(("step", "attn", "attn", "attn", "accept", "compact"))
    if op == "step":
        tree = rng.random() < 0.5
        new_hi = _log(rng, 1, 64) if tree else _log(rng, 1, 700)
        batch = _log(rng, 1, 512 if new_hi < 32 else 96 if tree else max(1, 16384 // new_hi))
        cached_hi = rng.choice((0, _log(rng, 1, 8000)))
        cols = rng.choice((16, 40, 160)) if cached_hi + new_hi <= 16 * BLOCK else 40
        return dict(op=op, batch=batch, cached_lo=rng.randint(0, cached_hi), cached_hi=cached_hi, new_lo=rng.randint(1, new_hi),
                    new_hi=new_hi, tree=tree, cols=cols)
    if op == "accept":
        hi = _log(rng, 1, 64)
        return dict(op=op, batch=_log(rng, 1, 512), new_lo=rng.randint(1, hi), new_hi=hi)
    if op == "compact":
        path, hi = rng.randint(2, 8), rng.randint(20, 64)
        ctx_hi = _log(rng, 65, 440)
        return dict(op=op, batch=_log(rng, 1, 100), ctx_lo=rng.randint(64, ctx_hi), ctx_hi=ctx_hi, new_lo=rng.randint(17, hi), new_hi=hi,
                    Hkv=rng.choice((1, 2)), path=path)
    H, Hkv = rng.choice(HEADS)
    hi, tree = _log(rng, 1, 128), rng.random() < 0.75
    ctx_hi = _log(rng, 200, 40960)
    most = 128 * 2300 * 8 * 64 * 32 // (8 * 32)      # token x node pairs of the largest case per kv head
    batch = _log(rng, 1, max(1, min(256, 128 * 2300 * 8 // (Hkv * ctx_hi), most * 8 // (ctx_hi * hi * H))))
    return dict(op=op, batch=batch, ctx_lo=rng.randint(hi, max(hi, ctx_hi)), ctx_hi=max(hi, ctx_hi), new_lo=rng.randint(1, hi), new_hi=hi,
                H=H, Hkv=Hkv, tree=tree)


# ---- inputs ----------------------------------------------------------------------------------------------------
def _spread(lo, hi, n):
    """n whole numbers, evenly over [lo, hi]."""
    return [lo + ((hi - lo) * i) // (n - 1) if n > 1 else (lo + hi + 1) // 2 for i in range(n)]


def _shuffled(values, g):
    t = torch.tensor(values, dtype=torch.int64)
    return t[torch.randperm(len(values), generator=g)]


def _cu(lens):
    return torch.cat([torch.zeros(1, dtype=torch.int64), lens.cumsum(0)])


def _parents(news, g):
    """Node 0 of each tree is its root; the parent of node j is any of the nodes before it."""
    j = torch.cat([torch.arange(int(n)) for n in news])
    p = (torch.rand(len(j), generator=g) * j).long().clamp(max=(j - 1).clamp(min=0))
    return torch.where(j > 0, p, -1)


def _tables(lens, g, blocks=0):
    """Block table rows for these lengths, ids scattered over a cache of `blocks`: (rows padded with -1, blocks in all)."""
    nb = (lens + BLOCK - 1) // BLOCK
    total = int(nb.sum())
    blocks = max(blocks, total + 3)
    ids = torch.randperm(blocks, generator=g)[:total]
    cols = max(1, int(nb.max()))
    at = torch.arange(cols)[None, :]
    where = at < nb[:, None]
    rows = torch.full((len(lens), cols), -1, dtype=torch.int64)
    rows[where] = ids
    return rows, blocks


def _i32(x):
    return x.to(torch.int32).to(DEV)


def prepare(case, seed):
    g = torch.Generator().manual_seed(seed)
    gd = torch.Generator(DEV).manual_seed(seed)
    b, op = case["batch"], case["op"]
    news = _shuffled(_spread(case["new_lo"], case["new_hi"], b), g)
    cu = _cu(news)
    total, words = int(cu[-1]), (int(news.max()) + 63) // 64
    s = dict(case=case, cu=_i32(cu), total=total, words=words, most=int(news.max()))
    if op == "step":
        cached = _shuffled(_spread(case["cached_lo"], case["cached_hi"], b), g)
        requests = b + 7
        rows = torch.randperm(requests, generator=g)[:b]
        held = (cached + BLOCK - 1) // BLOCK
        free = int(((news + BLOCK - 1) // BLOCK).sum()) + b + 11
        blocks = int(held.sum()) + free
        ids = torch.randperm(blocks, generator=g)
        tables = torch.full((requests, case["cols"]), -1, dtype=torch.int64)
        mine = torch.full((b, case["cols"]), -1, dtype=torch.int64)
        mine[torch.arange(case["cols"])[None, :] < held[:, None]] = ids[free:]
        tables[rows] = mine
        owned = torch.zeros(requests, dtype=torch.int64)
        owned[rows] = held
        stack = torch.zeros(blocks, dtype=torch.int64)
        stack[:free] = ids[:free]
        s.update(rows=_i32(rows), cached=_i32(cached), new=_i32(news), tables=_i32(tables), owned=_i32(owned), free=_i32(stack),
                 pool=_i32(torch.tensor([free, 0])), parents=_i32(_parents(news, g)) if case["tree"] else None)
    elif op == "attn":
        ctx = torch.maximum(_shuffled(_spread(case["ctx_lo"], case["ctx_hi"], b), g), news)
        rows, blocks = _tables(ctx, g)
        cache = lambda: torch.randn(blocks, BLOCK, case["Hkv"], D, generator=gd, device=DEV, dtype=torch.bfloat16)  # noqa: E731
        s.update(q=torch.randn(total, case["H"], D, generator=gd, device=DEV, dtype=torch.bfloat16), k=cache(), v=cache(), ctx=_i32(ctx),
                 bt=_i32(rows), masks=None, scale=D ** -0.5, most_ctx=int(ctx.max()))
        if case["tree"]:
            sees = _closure(_i32(_parents(news, g)), s["cu"], s["most"])
            s["masks"] = _pack(sees, words)[_flat(s["cu"], total)]
    elif op == "accept":
        parents = _parents(news, g)
        draft = torch.randint(0, VOCAB, (total,), generator=g)
        target = torch.randint(0, VOCAB, (total,), generator=g)
        # the target's sample is a drafted child's token at most nodes that have any
        first = cu[:-1].repeat_interleave(news)
        wanted = (torch.rand(total, generator=g) < 0.8) & (parents >= 0)
        child = torch.full((total,), -1, dtype=torch.int64)
        child.scatter_reduce_(0, (first + parents.clamp(min=0))[wanted], torch.arange(total)[wanted], "amax")
        target = torch.where(child >= 0, draft[child.clamp(min=0)], target)
        cached = torch.randint(1, 4000, (b,), generator=g)
        s.update(draft=draft.to(DEV), target=target.to(DEV), parents=_i32(parents), cached=_i32(cached), ctx=_i32(cached + news), path=min(16, s["most"]))
    else:
        # (the nodes that move lie behind all places they move to, so that a second pass moves the same values)
        n = case["path"]
        accepted = _shuffled(_spread(1, n, b), g)
        order = torch.rand(b, s["most"], generator=g)
        order[torch.arange(s["most"])[None, :] >= news[:, None]] = 2.0
        order[:, :n] = 2.0
        path = torch.cat([torch.zeros(b, 1, dtype=torch.int64), order.argsort(1)[:, :n - 1].sort(1).values], 1)
        path[torch.arange(n)[None, :] >= accepted[:, None]] = -1
        ctx = _shuffled(_spread(case["ctx_lo"], case["ctx_hi"], b), g)
        rows, blocks = _tables(ctx + news, g, int(((ctx + BLOCK - 1) // BLOCK).sum()) + b + 3)
        cache = torch.randn(2, LAYERS, blocks, BLOCK, case["Hkv"], D, generator=gd, device=DEV, dtype=torch.bfloat16)
        s.update(cache=cache, path=_i32(path), accepted=_i32(accepted), start=_i32(ctx), bt=_i32(rows))
    return s


# ---- plain forms -----------------------------------------------------------------------------------------------
def _flat(cu, total):
    """(sequence, place in it) of each token row."""
    t = torch.arange(total, device=cu.device)
    seq = torch.searchsorted(cu[1:].long(), t, right=True).clamp(max=len(cu) - 2)
    return seq, t - cu[seq].long()


def _padded(x, cu, most, fill):
    """Rows of each sequence as (batch, most, ...)."""
    at = cu[:-1].long()[:, None] + torch.arange(most, device=cu.device)[None, :]
    inside = at < cu[1:].long()[:, None]
    y = x[at.clamp(max=x.shape[0] - 1)]
    return torch.where(inside.reshape(inside.shape + (1,) * (y.dim() - 2)), y, fill)


def _closure(parents, cu, most):
    """(batch, most, most): node j sees node n, its ancestors and itself."""
    p = _padded(parents, cu, most, -1).long()
    sees = (p[:, :, None] == torch.arange(most, device=p.device)).float() + torch.eye(most, device=p.device)
    for _ in range(max(1, (most - 1).bit_length())):
        sees = (sees @ sees).clamp(max=1.0)
    return sees > 0


def _pack(sees, words):
    """Bits of (..., n) as (..., words) of 64, the lowest first."""
    bits = torch.nn.functional.pad(sees, (0, words * 64 - sees.shape[-1])).long()
    return (bits.reshape(*sees.shape[:-1], words, 64) << torch.arange(64, device=sees.device)).sum(-1)


def _plain_step(s):
    rows, cached, new, cu, total = s["rows"].long(), s["cached"].long(), s["new"].long(), s["cu"], s["total"]
    tables, owned, free, pool = s["tables"], s["owned"], s["free"], s["pool"]
    cols = tables.shape[1]
    cu_q = torch.nn.functional.pad(new.cumsum(0), (1, 0))
    held, need = owned[rows].long(), (cached + new + BLOCK - 1) // BLOCK
    fits = need <= cols
    want = torch.where(fits, (need - held).clamp(min=0), 0)
    upto = want.cumsum(0)
    ok = fits & ((want == 0) | (upto <= pool[0]))
    got = torch.where(ok, want, 0)
    at = torch.arange(cols, device=rows.device)[None, :]
    taken = (pool[0] - 1 - (upto - want))[:, None] - (at - held[:, None])
    fresh = (at >= held[:, None]) & (at < (held + got)[:, None])
    mine = torch.where(fresh, free[taken.clamp(0, len(free) - 1)], tables[rows])
    tables[rows] = mine
    owned[rows] = (held + got).int()
    pool[0] -= got.sum().int()
    context = torch.where(ok, cached + new, 0)
    cu_k = torch.nn.functional.pad(context.cumsum(0), (1, 0))
    block_tables = torch.where(ok[:, None] & (at < need[:, None]), mine, -1)
    seq, j = _flat(cu_q, total)
    pos = cached[seq] + j
    live = ok[seq]
    slot = torch.where(live, mine[seq, (pos // BLOCK).clamp(max=cols - 1)].long() * BLOCK + pos % BLOCK, -1)
    masks = None
    if s["parents"] is not None:
        sees = _closure(s["parents"], cu_q, s["most"])[seq, j]
        masks = torch.where(live[:, None], _pack(sees, s["words"]), 0)
        pos = cached[seq] + sees.sum(-1) - 1
    positions = torch.where(live, pos, 0)
    out = dict(cu_q=cu_q.int(), cu_k=cu_k.int(), context=context.int(), slots=slot.int(), positions=positions, tables=block_tables, masks=masks)
    # the step rolled back: each request keeps the blocks of its cached tokens
    keep = torch.minimum((cached + BLOCK - 1) // BLOCK, owned[rows].long())
    back = owned[rows].long() - keep
    before = back.cumsum(0) - back
    gone = (at >= keep[:, None]) & (at < (keep + back)[:, None])
    place = (pool[0] + back.sum() - 1 - before)[:, None] - (at - keep[:, None])
    current = tables[rows]
    # (what is not given back goes to a place behind the list)
    stack = torch.cat([free, free[:1]])
    stack[torch.where(gone, place, len(free))] = current
    free.copy_(stack[:-1])
    tables[rows] = torch.where(gone, -1, current)
    owned[rows] = keep.int()
    pool[0] += back.sum().int()
    return out


def _plain_attn(s):
    c, cu, total, most = s["case"], s["cu"], s["total"], s["most"]
    ctx, b, H, Hkv = s["ctx"].long(), c["batch"], c["H"], c["Hkv"]
    keys = torch.arange(s["most_ctx"], device=DEV)
    block = s["bt"].long()[:, keys // BLOCK].clamp(min=0)
    k, v = (s[n].view(-1, Hkv, D)[block * BLOCK + keys % BLOCK].float() for n in "kv")      # (batch, keys, kv heads, D)
    q = _padded(s["q"], cu, most, 0).float().view(b, most, Hkv, H // Hkv, D)
    score = torch.einsum("btkgd,bskd->bkgts", q, k) * s["scale"]
    news = (cu[1:] - cu[:-1]).long()
    node = keys[None, :] - (ctx - news)[:, None]                                            # (batch, keys)
    place = torch.arange(most, device=DEV)
    if s["masks"] is None:
        drafted = node[:, None, :] <= place[None, :, None]
    else:
        word = _padded(s["masks"], cu, most, 0)                                             # (batch, nodes, words)
        which = node.clamp(0, 64 * s["words"] - 1)
        drafted = (word.gather(2, (which // 64)[:, None, :].expand(-1, most, -1)) >> (which % 64)[:, None, :] & 1) == 1
    sees = (node < 0)[:, None, :] | (drafted & (node >= 0)[:, None, :])
    sees = (sees & (keys[None, :] < ctx[:, None])[:, None, :])[:, None, None]
    score = score.masked_fill(~sees, float("-inf"))
    weight = torch.exp(score - score.amax(-1, keepdim=True).clamp(min=-1e30))
    weight = weight / weight.sum(-1, keepdim=True).clamp(min=1e-30)
    out = torch.einsum("bkgts,bskd->btkgd", weight, v).reshape(b, most, H, D)
    return out[_flat(cu, total)].to(torch.bfloat16)


def _plain_accept(s):
    cu, total, most, n = s["cu"], s["total"], s["most"], s["path"]
    parents = _padded(s["parents"], cu, most, -1).long()
    draft, target = _padded(s["draft"], cu, most, -1), _padded(s["target"], cu, most, -2)
    hit = (parents >= 0) & (draft == target.gather(1, parents.clamp(min=0)))
    place = torch.arange(most, device=DEV)
    # of the children that hit, a node is followed by the one of lowest index
    rival = hit[:, None, :] & (parents[:, None, :] == parents[:, :, None]) & (place[None, :] < place[:, None])
    chosen = (hit & ~rival.any(-1)) | (place == 0)
    sees = _closure(s["parents"], cu, most)
    on = (~sees | chosen[:, None, :]).all(-1) & sees[:, :, 0] & (place[None, :] < (cu[1:] - cu[:-1])[:, None])
    depth = on.cumsum(1) - 1
    on = on & (depth < n)
    accepted = on.sum(1)
    path = torch.full((len(cu) - 1, n + 1), -1, device=DEV, dtype=torch.int64)
    path.scatter_(1, torch.where(on, depth, n), torch.where(on, place, -1))
    path = path[:, :n]
    tokens = torch.where(path >= 0, target.gather(1, path.clamp(min=0)), -1)
    return dict(accepted=accepted.int(), path=path.int(), tokens=tokens, cached=(s["cached"] + accepted).int())


def _plain_compact(s):
    cache, path, start, n = s["cache"], s["path"].long(), s["start"].long()[:, None], s["path"].shape[1]
    to = torch.arange(n, device=DEV)[None, :]
    to = torch.where(path >= 0, to, 0)                   # (what is not accepted: the root onto itself)
    at = torch.stack([start + path.clamp(min=0), start + to])
    block = s["bt"].long()[torch.arange(len(path), device=DEV)[None, :, None], at // BLOCK]
    src, dst = (block * BLOCK + at % BLOCK).reshape(2, -1)
    rows = cache.view(-1, cache.shape[2] * BLOCK, cache.shape[4] * D)
    rows[:, dst] = rows[:, src]
    return cache


# ---- the framework's operators ---------------------------------------------------------------------------------
def _own(s):
    op = s["case"]["op"]
    if op == "attn":
        from nanovllm_b200 import tree_attention
        return tree_attention(s["q"], s["k"], s["v"], s["cu"], s["ctx"], s["bt"], s["masks"], s["scale"], s["case"]["Hkv"])
    if op == "step":
        from nanovllm_b200.engine.block_tables import DeviceBlockTables
        state = DeviceBlockTables(s["tables"], s["owned"], s["free"], s["pool"], BLOCK)
        t = state.step(s["rows"], s["cached"], s["new"], s["total"], s["parents"], s["words"] if s["parents"] is not None else 0)
        state.release(s["rows"], s["cached"])
        return dict(cu_q=t.cu_seqlens_q, cu_k=t.cu_seqlens_k, context=t.context_lens, slots=t.slot_mapping, positions=t.positions,
                    tables=t.block_tables, masks=t.tree_masks)
    from nanovllm_b200.engine.tree_decode import accept_tree, compact_kvcache
    if op == "accept":
        t = accept_tree(s["draft"], s["target"], s["parents"], s["cu"], s["cached"], s["ctx"], s["path"])
        return dict(accepted=t.accepted, path=t.path, tokens=t.tokens, cached=t.cached_lens)
    compact_kvcache(s["cache"], s["path"], s["accepted"], s["start"], s["bt"])
    return s["cache"]


def run(state):
    op = state["case"]["op"]
    if own:
        out = _own(state)
    elif op == "attn":
        out = _plain_attn(state)
    elif op == "step":
        out = _plain_step(state)
    elif op == "accept":
        out = _plain_accept(state)
    else:
        out = _plain_compact(state)
    if op == "step":
        # the allocator's state after the roll-back
        out.update(request_tables=state["tables"], owned=state["owned"], free=state["free"], pool=state["pool"])
    return out


def work(case):
    b, op = case["batch"], case["op"]
    news = _spread(case["new_lo"], case["new_hi"], b)
    total = sum(news)
    if op == "step":
        cached = _spread(case["cached_lo"], case["cached_hi"], b)
        words = (max(news) + 63) // 64 if case["tree"] else 0
        fresh = sum(max(0, -(-(c + n) // BLOCK) - -(-c // BLOCK)) for c, n in zip(cached, news))
        held = sum(-(-c // BLOCK) for c in cached)
        # lengths, held ids and parents in; tables, slots, positions and masks out; taken ids out of the list and back into it
        return dict(bytes=b * 32 + held * 4 + b * case["cols"] * 4 + total * (12 + 8 * words + (4 if case["tree"] else 0)) + fresh * 20, flops=0)
    if op == "accept":
        return dict(bytes=total * 20 + b * (16 + 12 * min(16, max(news))), flops=0)
    if op == "compact":
        moved = sum(_spread(1, case["path"], b)) - b
        return dict(bytes=2 * moved * 2 * LAYERS * case["Hkv"] * D * 2 + b * (8 + 4 * case["path"]), flops=0)
    ctx = [max(c, min(news)) for c in _spread(case["ctx_lo"], case["ctx_hi"], b)]
    words = (max(news) + 63) // 64 if case["tree"] else 0
    pairs = sum(ctx) * total / b                          # (lengths and tree sizes are shuffled apart)
    return dict(bytes=sum(ctx) * case["Hkv"] * D * 4 + total * (case["H"] * D * 4 + 8 * words) + -(-sum(ctx) // BLOCK) * 4,
                flops=4 * D * case["H"] * pairs)


# ---- the definition, in 64 bits --------------------------------------------------------------------------------
def exact(case, seed):
    if case["op"] not in ("attn", "compact"):
        return None                                       # whole numbers
    s = prepare(case, seed)
    table, cu = s["bt"].tolist(), s["cu"].tolist()
    if case["op"] == "compact":
        cache, before = s["cache"], s["cache"].clone()
        for i, (path, start) in enumerate(zip(s["path"].tolist(), s["start"].tolist())):
            for k, node in enumerate(path):
                if node >= 0:
                    old, new = start + node, start + k
                    cache[:, :, table[i][new // BLOCK], new % BLOCK] = before[:, :, table[i][old // BLOCK], old % BLOCK]
        return cache
    G = case["H"] // case["Hkv"]
    out = torch.zeros(s["total"], case["H"], D, dtype=torch.float64, device=DEV)
    for i, n in enumerate(s["ctx"].tolist()):
        lo, hi = cu[i], cu[i + 1]
        blocks = torch.tensor(table[i][: -(-n // BLOCK)], device=DEV)
        k, v = (s[x][blocks].reshape(-1, case["Hkv"], D)[:n].double() for x in "kv")
        seen = torch.ones(hi - lo, n, dtype=torch.bool, device=DEV)
        if s["masks"] is None:
            seen[:, n - (hi - lo):] = torch.tril(seen[:, n - (hi - lo):])
        else:
            bits = torch.stack([(s["masks"][lo:hi, j // 64] >> (j % 64)) % 2 != 0 for j in range(hi - lo)], 1)
            seen[:, n - (hi - lo):] = bits
        for h in range(case["H"]):
            x = s["q"][lo:hi, h].double() @ k[:, h // G].T * s["scale"]
            out[lo:hi, h] = torch.softmax(x.masked_fill(~seen, -math.inf), 1) @ v[:, h // G]
    return out
