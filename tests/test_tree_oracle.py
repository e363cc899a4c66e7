"""CPU: the plain restatement of a step with drafted trees (oracle/tree_oracle.py) against the oracles of decode, prefill, store and
metadata, which are pinned to the reference's own outputs, and against definitions written another way."""
import random

import pytest
import torch

from oracle.attention_oracle import _gather_paged, decode_attn_ref, prefill_attn_ref, store_kvcache_ref
from oracle.metadata_oracle import prepare_decode_ref
from oracle.tree_oracle import BlockState, accept_tree_ref, compact_ref, tree_attn_ref
from test_decode_metadata import FakeSeq
from test_tree_decode import attention_case, random_parents


def close(a, b, weight):
    """`a` has been rounded to bf16 (2^-8 of itself at most) from sums in 32 bits (scores of 128 products, up to 300 keys: below
    2^-14 of sum p |v| together)."""
    a, b = a.double(), b.double()
    assert bool(((a - b).abs() <= 2.0 ** -8 * b.abs() + 2.0 ** -14 * weight).all())


@pytest.mark.parametrize("H,hkv", [(4, 2), (8, 1), (3, 3)])
def test_one_node_is_decode(H, hkv):
    ctx = [1, 5, 256, 257, 300, 0]
    c = attention_case(H, hkv, ctx, [1] * 6, seed=H, masks="chain", poison=False)
    out, weight = tree_attn_ref(c["q"], c["k"], c["v"], c["cu"], ctx, c["tables"], None, c["scale"])
    close(decode_attn_ref(c["q"], c["k"], c["v"], torch.tensor(ctx), torch.tensor(c["tables"], dtype=torch.int64), c["scale"]).view(-1, H, 128), out, weight)
    ones = torch.ones(6, 1, dtype=torch.int64)
    assert torch.equal(tree_attn_ref(c["q"], c["k"], c["v"], c["cu"], ctx, c["tables"], ones, c["scale"])[0], out)


@pytest.mark.parametrize("H,hkv", [(4, 2), (2, 1)])
def test_a_chain_is_the_end_of_a_prefill(H, hkv):
    ctx, nodes = [70, 300, 65, 3, 130], [5, 33, 65, 1, 70]
    cu_k = [0]
    for n in ctx:
        cu_k.append(cu_k[-1] + n)
    c = attention_case(H, hkv, ctx, nodes, seed=H + 9, masks="chain", poison=False)
    out, weight = tree_attn_ref(c["q"], c["k"], c["v"], c["cu"], ctx, c["tables"], None, c["scale"])
    tables = torch.tensor(c["tables"], dtype=torch.int64)
    close(prefill_attn_ref(c["q"], c["k"], c["v"], torch.tensor(c["cu"]), torch.tensor(cu_k), c["scale"], tables), out, weight)
    # the same chain by its masks: node j sees nodes 0 .. j
    bits = [[(1 << min(max(j + 1 - 64 * w, 0), 64)) - 1 for w in range(2)] for n in nodes for j in range(n)]
    masks = torch.tensor([[b - 2 ** 64 if b >> 63 else b for b in row] for row in bits], dtype=torch.int64)
    assert torch.equal(tree_attn_ref(c["q"], c["k"], c["v"], c["cu"], ctx, c["tables"], masks, c["scale"])[0], out)


def test_a_node_is_decode_along_its_ancestors():
    """Each node's row is single-token decode over a cache that holds the context and the node's path, one behind the other."""
    rng, H, hkv, ctx, nodes = random.Random(2), 4, 2, [20, 90], [9, 70]
    c = attention_case(H, hkv, ctx, nodes, seed=3, poison=False)
    parents = [[-1] + [rng.randrange(j) for j in range(1, n)] for n in nodes]
    paths, rows = [], []
    for p in parents:
        for j in range(len(p)):
            path = [j]
            while p[path[-1]] >= 0:
                path.append(p[path[-1]])
            paths.append(path[::-1])
            mask = sum(1 << x for x in path)
            rows.append([w - 2 ** 64 if w >> 63 else w for w in (mask & (2 ** 64 - 1), mask >> 64)])
    out, weight = tree_attn_ref(c["q"], c["k"], c["v"], c["cu"], ctx, c["tables"], torch.tensor(rows, dtype=torch.int64), c["scale"])
    for r, path in enumerate(paths):
        i = 0 if r < nodes[0] else 1
        front = ctx[i] - nodes[i]
        seen = list(range(front)) + [front + x for x in path]
        table = torch.tensor(c["tables"][i], dtype=torch.int64)
        line = [torch.zeros(1, 256, hkv, 128, dtype=torch.bfloat16) for _ in range(2)]
        for own, cache in zip(line, (c["k"], c["v"])):
            own[0, :len(seen)] = _gather_paged(cache, table, ctx[i], 256)[seen]
        close(decode_attn_ref(c["q"][r:r + 1], *line, torch.tensor([len(seen)]), torch.zeros(1, 1, dtype=torch.int64), c["scale"])[:, 0], out[r:r + 1], weight[r:r + 1])


def test_a_decode_step_is_what_the_model_runner_prepares():
    rng, bs = random.Random(4), 256
    state = BlockState([[-1] * 8 for _ in range(40)], [0] * 40, rng.sample(range(400), 400), bs)
    lens = [rng.choice((1, 255, 256, 257, rng.randint(1, 1500))) for _ in range(40)]
    state.step(None, [0] * 40, lens, sum(lens))
    for _ in range(3):
        order = rng.sample(range(40), 33)
        s = state.step(order, [lens[r] for r in order], [1] * 33, 33)
        seqs = [FakeSeq(lens[r] + 1, state.tables[r][:state.owned[r]], 7) for r in order]
        _, positions, slots, context, tables = prepare_decode_ref(seqs, bs)
        assert s["positions"] == positions.tolist() and s["slots"] == slots.tolist() and s["ctx"] == context.tolist()
        assert [row[:tables.size(1)] for row in s["tables"]] == tables.tolist() and all(x == -1 for row in s["tables"] for x in row[tables.size(1):])
        assert s["cu_q"] == list(range(34)) and s["cu_k"][-1] == sum(s["ctx"])
        for r in order:
            lens[r] += 1
    # every block is in one place
    held = [b for r in range(40) for b in state.tables[r][:state.owned[r]]]
    assert sorted(held + state.free) == list(range(400))


def test_a_step_stores_where_its_tables_read_and_gives_back_what_it_took():
    rng, bs = random.Random(5), 256
    state = BlockState([[-1] * 4 for _ in range(5)], [0] * 5, rng.sample(range(30), 30), bs)
    cached, new = [0, 250, 256, 3, 700], [300, 10, 1, 0, 64]
    state.step(None, [0] * 5, cached, sum(cached))
    before = ([list(r) for r in state.tables], list(state.owned), list(state.free))
    parents = random_parents(new, rng, chain=True)
    s = state.step(None, cached, new, sum(new), parents, 5)
    assert not state.left_out
    rows = torch.arange(1, sum(new) + 1, dtype=torch.float32).view(-1, 1, 1).expand(-1, 1, 2).contiguous()
    cache = [torch.zeros(30, bs, 1, 2) for _ in range(2)]
    store_kvcache_ref(rows, rows, *cache, torch.tensor(s["slots"]))
    for i in range(5):
        got = _gather_paged(cache[0], torch.tensor(s["tables"][i]), s["ctx"][i], bs)[cached[i]:, 0, 0].tolist()
        assert got == list(range(s["cu_q"][i] + 1, s["cu_q"][i + 1] + 1)) and s["ctx"][i] == cached[i] + new[i]
        # of a chain: positions one behind the other, each sees those before it
        assert s["positions"][s["cu_q"][i]:s["cu_q"][i + 1]] == list(range(cached[i], cached[i] + new[i]))
    for i in range(5):
        for j in range(new[i]):
            assert sum((w % 2 ** 64) << (64 * x) for x, w in enumerate(s["masks"][s["cu_q"][i] + j])) == (1 << (j + 1)) - 1
    state.release(None, cached)
    assert (state.tables, state.owned, state.free) == before


def test_masks_are_the_closure_of_the_parents():
    rng, n = random.Random(6), 100
    parents = random_parents([n], rng)
    s = BlockState([[-1]], [0], [0], 256).step(None, [5], [n], n, parents, 2)
    sees = torch.eye(n, dtype=torch.bool)
    for j in range(1, n):
        sees[j] |= sees[parents[j]]
    for j in range(n):
        assert [(s["masks"][j][x // 64] >> (x % 64)) & 1 for x in range(n)] == sees[j].int().tolist()
        assert s["positions"][j] == 5 + int(sees[j].sum()) - 1


@pytest.mark.parametrize("vocab", [1, 2, 3])
def test_the_walk_follows_the_first_child_that_was_sampled(vocab):
    rng = random.Random(vocab)
    for _ in range(30):
        n, most = rng.randint(1, 30), rng.randint(1, 8)
        parents, draft, target = random_parents([n], rng), [rng.randrange(vocab) for _ in range(n)], [rng.randrange(vocab) for _ in range(n)]
        accepted, path, tokens, lens = accept_tree_ref(draft, target, parents, [0, n], [11], [11 + n], most)
        p = path[0][:accepted[0]]
        assert p[0] == 0 and 1 <= len(p) <= most and lens == [11 + len(p)] and path[0][len(p):] == [-1] * (most - len(p))
        first = lambda cur: next((c for c in range(n) if c > cur and parents[c] == cur and draft[c] == target[cur]), None)  # noqa: E731
        assert all(first(a) == b for a, b in zip(p, p[1:])) and (len(p) == most or first(p[-1]) is None)
        # what comes out is what the target sampled: each accepted draft is the token in front of it
        assert tokens[0][:len(p)] == [target[x] for x in p] and [draft[x] for x in p[1:]] == tokens[0][:len(p) - 1]
    assert accept_tree_ref([1], [1], [-1], [0, 1], [4], [0], 2)[0] == [0]


def test_the_moves_leave_the_accepted_path_in_line():
    rng, bs = random.Random(8), 4
    table = rng.sample(range(12), 10)
    cache = torch.arange(2 * 12 * bs, dtype=torch.int64).view(2, 12, bs)
    path, start = [0, 2, 3, 7, 20], 6
    want = [[cache[p, table[(start + x) // bs], (start + x) % bs].item() for x in path] for p in range(2)]
    front = [[cache[p, table[x // bs], x % bs].item() for x in range(start)] for p in range(2)]
    compact_ref(cache, [path + [-1]], [5], [start], [table], bs)
    line = lambda p, a, b: [cache[p, table[x // bs], x % bs].item() for x in range(a, b)]  # noqa: E731
    assert [line(p, start, start + 5) for p in range(2)] == want and [line(p, 0, start) for p in range(2)] == front
