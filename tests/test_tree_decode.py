"""A step with drafted trees: tables from request lengths, attention of the nodes over the cache, the walk along the sampled
tokens, the moves in the cache, and a run of them together.  Whole numbers and moved rows are compared exactly.

Attention: probabilities are rounded to bf16 in front of the product with V (each off by 2^-8 of itself at most), and so is the
output; sums, maxima and scores have 32 bits, and their errors together are below 2^-11 here (a score of 128 products of size
up to 5 is off by 129 * 2^-24 * scale * sum |q||k| < 2^-13, exp2 by 2^-22).  With A = sum p |v| that is
|error| <= (2^-8 + 2^-11) * (A + |out|)."""
import random

import pytest
import torch

import nanovllm_b200
from nanovllm_b200 import _lib
from nanovllm_b200.engine.block_tables import DeviceBlockTables, StepTables
from nanovllm_b200.engine.tree_decode import accept_tree, compact_kvcache
from oracle.tree_oracle import BlockState, accept_tree_ref, compact_ref, tree_attn_ref
from test_early_start import _compare, late_copy  # noqa: F401  (late_copy is a fixture)

DEV = "cuda:0"
BOUND = 2.0 ** -8 + 2.0 ** -11


def i32(x, dev=DEV):
    return torch.tensor(x, dtype=torch.int32, device=dev)


def i64(x, dev=DEV):
    return torch.tensor(x, dtype=torch.int64, device=dev)


def status_ok():
    _lib.check(_lib.load().b200_device_status())


def random_parents(news, rng, chain=False):
    out = []
    for n in news:
        out += [-1 if j == 0 else j - 1 if chain else rng.randrange(j) for j in range(n)]
    return out


# ---- refusals (no GPU) -----------------------------------------------------------------------------------------
def test_c_entries_refuse_without_a_device(lib):
    step = lambda **k: lib.b200_step_tables(*{**dict(  # noqa: E731
        rows=None, cached=16, new=16, parents=None, batch=1, tokens=4, bs=256, tables=16, stride=4, cols=4, requests=1, owned=16, free=16,
        pool=16, blocks=8, buffer=1, cu_q=16, cu_k=16, ctx=16, slots=16, pos=16, bt=16, masks=None, words=0, stream=None), **k}.values())
    assert step(batch=-1) == -2 and step(batch=4097, buffer=4097) == -2 and step(buffer=0) == -2 and step(tokens=-1) == -2
    assert step(bs=128) == -2 and step(blocks=0) == -2 and step(blocks=1 << 23) == -2 and step(cols=0) == -2 and step(stride=3) == -2
    assert step(cols=1 << 19, stride=1 << 19) == -2
    for name in ("cached", "new", "tables", "owned", "free", "pool", "cu_q", "cu_k", "ctx", "slots", "pos", "bt"):
        assert step(**{name: None}) == -1, name
    assert step(parents=16) == -1 and step(masks=16, words=1) == -1
    assert step(parents=16, masks=16, words=5) == -2 and step(parents=16, masks=16, words=0) == -2
    assert step(parents=16, masks=20, words=1) == -3 and step(pos=20) == -3
    rel = lambda **k: lib.b200_release_blocks(*{**dict(  # noqa: E731
        rows=None, keep=16, batch=1, bs=256, tables=16, stride=4, cols=4, requests=1, owned=16, free=16, pool=16, blocks=8, stream=None), **k}.values())
    assert rel(batch=0) == 0 and rel(batch=5000) == -2 and rel(keep=None) == -1 and rel(tables=None) == -1 and rel(bs=100) == -2
    tree = lambda **k: lib.b200_tree_attn(*{**dict(  # noqa: E731
        q=16, qs=2048, k=16, v=16, blocks=8, bs=256, bt=16, bts=4, cols=4, cu=16, ctx=16, masks=None, words=0, out=16, ws=16, wsb=1 << 40,
        batch=1, total=4, H=16, Hkv=8, D=128, scale=0.1, stream=None), **k}.values())
    assert tree(batch=0) == 0 and tree(total=0) == 0 and tree(batch=-1) == -2 and tree(D=64) == -2 and tree(Hkv=5) == -2 and tree(H=1032, qs=1032 * 128) == -2
    assert tree(masks=16, words=5) == -2 and tree(masks=16, words=0) == -2 and tree(bs=200) == -2 and tree(blocks=0) == -2 and tree(cols=0) == -2 and tree(bts=3) == -2
    assert tree(cols=1 << 22, bts=1 << 22) == -2
    for name in ("q", "k", "v", "bt", "cu", "ctx", "out"):
        assert tree(**{name: None}) == -1, name
    assert tree(q=24) == -3 and tree(qs=2047) == -3 and tree(qs=1024) == -3 and tree(out=24) == -3 and tree(masks=20, words=1) == -3
    assert tree(ws=None) in (-4, -5) and tree(wsb=0) in (-4, -5)
    assert lib.b200_tree_workspace_bytes(16, 5, 128) == -2 and lib.b200_tree_workspace_bytes(16, 8, 64) == -2
    acc = lambda **k: lib.b200_accept_tree(*{**dict(  # noqa: E731
        draft=16, target=16, parents=16, cu=16, cached=16, ctx=16, batch=1, tokens=4, path=4, accepted=16, p=16, out=16, lens=16, stream=None), **k}.values())
    assert acc(batch=0) == 0 and acc(batch=-1) == -2 and acc(path=0) == -2 and acc(tokens=-1) == -2 and acc(draft=20) == -3 and acc(out=20) == -3
    for name in ("draft", "target", "parents", "cu", "cached", "ctx", "accepted", "p", "out", "lens"):
        assert acc(**{name: None}) == -1, name
    com = lambda **k: lib.b200_compact_kvcache(*{**dict(  # noqa: E731
        cache=16, planes=2, stride=1 << 20, row=256, blocks=4, bs=256, path=16, cols=4, accepted=16, start=16, bt=16, bts=4, btc=4, batch=1, stream=None), **k}.values())
    assert com(batch=0) == 0 and com(planes=0) == 0 and com(cols=1) == 0 and com(batch=65536) == -2 and com(row=0) == -2 and com(stride=1 << 17) == -2
    assert com(row=264, stride=1 << 20) == -3 and com(cache=20) == -3 and com(stride=(1 << 20) + 8) == -3 and com(btc=5) == -2
    for name in ("cache", "path", "accepted", "start", "bt"):
        assert com(**{name: None}) == -1, name


def test_python_entries_refuse_cpu_tensors_and_wrong_types():
    z = lambda *s, t=torch.int32: torch.zeros(*s, dtype=t)  # noqa: E731
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        nanovllm_b200.tree_attention(z(1, 16, 128, t=torch.bfloat16), z(1, 256, 8, 128, t=torch.bfloat16), z(1, 256, 8, 128, t=torch.bfloat16),
                                     z(2), z(1), z(1, 1), None, 0.1, 8)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        DeviceBlockTables(z(1, 1), z(1), z(1), z(2), 256).step(None, z(1), z(1), 0)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        DeviceBlockTables(z(1, 1), z(1), z(1), z(2), 256).release(None, z(1))
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        accept_tree(z(1, t=torch.int64), z(1, t=torch.int64), z(1), z(2), z(1), z(1), 1)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        compact_kvcache(z(2, 1, 256, 1, 128, t=torch.bfloat16), z(1, 2), z(1), z(1), z(1, 1))
    with pytest.raises(TypeError, match="tree_masks"):
        nanovllm_b200.tree_attention(z(1, 16, 128, t=torch.bfloat16), z(1, 256, 8, 128, t=torch.bfloat16), z(1, 256, 8, 128, t=torch.bfloat16),
                                     z(2), z(1), z(1, 1), 3, 0.1, 8)


@pytest.mark.gpu
def test_python_entries_refuse_on_the_gpu():
    z = lambda *s, t=torch.int32: torch.zeros(*s, dtype=t, device=DEV)  # noqa: E731
    bf = torch.bfloat16
    q, c, cu, ctx, bt = z(4, 16, 128, t=bf), z(2, 256, 8, 128, t=bf), z(2), z(1), z(1, 2)
    call = lambda q=q, k=c, v=c, cu=cu, ctx=ctx, bt=bt, m=None, s=0.1, h=8: nanovllm_b200.tree_attention(q, k, v, cu, ctx, bt, m, s, h)  # noqa: E731
    assert call().shape == (4, 16, 128)
    for bad in (dict(q=q.half()), dict(k=c.half()), dict(h=4), dict(v=c[:1]), dict(k=c.transpose(0, 1)), dict(cu=cu.long()), dict(cu=z(3)),
                dict(bt=bt.long()), dict(bt=z(0, 2)), dict(m=z(4, 1)), dict(m=z(3, 1, t=torch.int64)), dict(m=z(4, 5, t=torch.int64)),
                dict(q=z(4, 128, 16, t=bf).transpose(1, 2)), dict(ctx=ctx.cpu().cuda().float()), dict(bt=z(2, 1).t()[:, ::2].expand(1, 2))):
        with pytest.raises(AssertionError):
            call(**bad)
    with pytest.raises(ValueError):
        call(q=z(4, 2048, t=bf))
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        call(ctx=ctx.cpu())
    for bad in (dict(q=z(4, 16, 64, t=bf), k=z(2, 256, 8, 64, t=bf), v=z(2, 256, 8, 64, t=bf)), dict(k=z(2, 128, 8, 128, t=bf), v=z(2, 128, 8, 128, t=bf)),
                dict(m=z(4, 0, t=torch.int64)), dict(q=z(4, 12, 128, t=bf))):
        with pytest.raises(_lib.B200AttnError):
            call(**bad)
    state = DeviceBlockTables.create(4, 3, 8, 256, DEV)
    for args in ((None, z(2), z(3), 0), (None, z(5), z(5), 0), (z(1), z(2), z(2), 0), (None, z(2).long(), z(2), 0), (None, z(2), z(2), -1),
                 (None, z(2), z(2), 4, z(3), 1), (None, z(2), z(2), 4, z(4), 0), (None, z(2), z(2), 4, z(4), 5), (None, z(2), z(2), 4, None, 1)):
        with pytest.raises(AssertionError):
            state.step(*args)
    with pytest.raises(AssertionError):
        state.step(None, z(2), z(2), 4, out=StepTables(z(3), z(3), z(2), z(5), z(4, t=torch.int64), z(2, 3), None))
    with pytest.raises(AssertionError):
        state.release(z(2), z(3))
    with pytest.raises(AssertionError):
        accept_tree(z(4), z(4, t=torch.int64), z(4), z(2), z(1), z(1), 4)
    with pytest.raises(AssertionError):
        accept_tree(z(4, t=torch.int64), z(4, t=torch.int64), z(4), z(2), z(1), z(1), 0)
    kv = z(2, 2, 2, 256, 1, 128, t=bf)
    for args in ((kv.transpose(0, 1), z(1, 2), z(1), z(1), z(1, 1)), (kv, z(2, 2), z(1), z(1), z(1, 1)), (kv, z(1, 2), z(1), z(2), z(1, 1)),
                 (kv, z(1, 2), z(1), z(1), z(0, 1)), (kv, z(1, 2).long(), z(1), z(1), z(1, 1))):
        with pytest.raises(AssertionError):
            compact_kvcache(*args)
    status_ok()


# ---- tables ----------------------------------------------------------------------------------------------------
def device_state(ref, blocks):
    free = ref.free + [-7] * (blocks - len(ref.free))
    return DeviceBlockTables(i32(ref.tables), i32(ref.owned), i32(free), i32([len(ref.free), 0]), ref.block_size)


def same_state(dev, ref):
    n = len(ref.free)
    assert dev.pool.tolist() == [n, ref.left_out]
    assert dev.free_blocks.tolist()[:n] == ref.free
    assert dev.owned.tolist() == ref.owned and dev.tables.tolist() == ref.tables


def same_step(got, want, words):
    assert got.cu_seqlens_q.tolist() == want["cu_q"] and got.cu_seqlens_k.tolist() == want["cu_k"]
    assert got.context_lens.tolist() == want["ctx"] and got.slot_mapping.tolist() == want["slots"]
    assert got.positions.tolist() == want["positions"]
    assert got.block_tables.tolist()[:len(want["tables"])] == want["tables"]
    if words:
        assert got.tree_masks.tolist() == want["masks"]
    else:
        assert got.tree_masks is None


@pytest.mark.gpu
@pytest.mark.parametrize("batch,cols,bs,words,seed", [(1, 1, 256, 0, 0), (1, 3, 256, 1, 1), (7, 5, 512, 2, 2), (33, 4, 256, 0, 3), (65, 9, 256, 4, 4),
                                                      (513, 3, 256, 1, 5), (1025, 2, 256, 0, 6), (4096, 2, 256, 1, 7), (300, 160, 256, 1, 8)])
def test_step_tables_over_several_steps(batch, cols, bs, words, seed):
    """Growing sequences, in a new order each step, some of them rolled back, against the lists."""
    rng = random.Random(seed)
    requests = batch + 3
    blocks = requests * min(cols, 5) + 2
    ids = list(range(blocks))
    rng.shuffle(ids)
    ref = BlockState([[-1] * cols for _ in range(requests)], [0] * requests, ids, bs)
    dev = device_state(ref, blocks)
    lens = [0] * requests
    for step in range(4):
        rows = rng.sample(range(requests), batch)
        room = min(cols, 5) * bs
        new = [min(rng.choice((0, 1, 1, 5, 64 * words if words else 300, rng.randint(1, 64 * words if words else 700))), room - lens[r]) for r in rows]
        cached = [lens[r] for r in rows]
        total = sum(new)
        parents = random_parents(new, rng, chain=step == 2) if words else None
        want = ref.step(rows, cached, new, total, parents, words)
        got = dev.step(i32(rows), i32(cached), i32(new), total, i32(parents) if words else None, words)
        same_step(got, want, words)
        same_state(dev, ref)
        assert dev.pool[1] == 0
        keep = [lens[r] + rng.randint(0, n) for r, n in zip(rows, new)]
        for r, k in zip(rows, keep):
            lens[r] = k
        ref.release(rows, keep)
        dev.release(i32(rows), i32(keep))
        same_state(dev, ref)
    status_ok()


@pytest.mark.gpu
def test_step_tables_leave_out_what_cannot_be_served():
    """Rows outside the range, named twice, too long for the table or the mask, out of blocks, out of token rows."""
    bs, cols = 256, 4
    ref = BlockState([[-1] * cols for _ in range(12)], [0] * 12, list(range(9, -1, -1)), bs)
    ref.tables[5][:2], ref.owned[5] = [20, 21], 2
    blocks = 24
    dev = device_state(ref, blocks)
    rows = [3, -1, 12, 3, 5, 6, 7, 8, 9, 10, 5, 11, 0]
    cached = [0, 0, 0, 0, 500, 0, 1000, 700, 0, 100, 0, -5, 0]
    new = [300, 5, 5, 7, 10, 0, 25, 64, 700, 60, 1, -3, 2]
    for words in (0, 1):
        parents = random_parents([max(n, 0) for n in new], random.Random(1)) if words else None
        total = sum(max(n, 0) for n in new) - 1                     # the last sequence's tokens do not fit
        want = ref.step(rows, cached, new, total, parents[:total] if words else None, words, buffer_rows=16)
        out = StepTables(i32([9] * 17), i32([9] * 17), i32([9] * 16), i32([9] * total), i64([9] * total), i32([[9] * cols] * 16),
                         i64([[9] * words] * total) if words else None)
        got = dev.step(i32(rows), i32(cached), i32(new), total, i32(parents[:total]) if words else None, words, out=out)
        same_step(got, want, words)
        assert got.context_lens.data_ptr() == out.context_lens.data_ptr() and got.block_tables[13:].eq(9).all()
        same_state(dev, ref)
        assert ref.left_out >= 6
    # nothing is left: a sequence that needs a block is left out, one that does not is served
    ref.free = []
    dev = device_state(ref, blocks)
    want = ref.step([0, 5], [0, 505], [1, 7], 8)
    got = dev.step(i32([0, 5]), i32([0, 505]), i32([1, 7]), 8)
    same_step(got, want, 0)
    same_state(dev, ref)
    assert want["ctx"] == [0, 512]
    # the same row twice, rows outside, lengths beyond what is held and below zero
    rows, keep = [5, 5, -1, 12, 3, 7], [300, 0, 0, 0, -9, 10 ** 9]
    ref.release(rows, keep)
    dev.release(i32(rows), i32(keep))
    same_state(dev, ref)
    # a batch of none, tokens of none
    got = dev.step(i32([]), i32([]), i32([]), 3)
    assert got.cu_seqlens_q.tolist() == [0] and got.slot_mapping.tolist() == [-1] * 3 and got.positions.tolist() == [0] * 3
    got = dev.step(None, i32([0, 0]), i32([0, 0]), 0)
    assert got.cu_seqlens_q.tolist() == [0, 0, 0] and got.context_lens.tolist() == [0, 0]
    dev.release(None, i32([]))
    status_ok()


# ---- attention -------------------------------------------------------------------------------------------------
def attention_case(H, hkv, ctx, nodes, seed, masks="tree", words=None, bs=256, extra_rows=0, poison=True):
    """Inputs on the CPU.  Slots that no sequence owns hold NaN, table tails stale ids."""
    rng, g = random.Random(seed), torch.Generator().manual_seed(seed)
    need = [-(-max(c, 0) // bs) for c in ctx]
    cols = max(need + [1]) + 1
    blocks = sum(need) + 2
    ids = list(range(blocks))
    rng.shuffle(ids)
    k = torch.randn(blocks, bs, hkv, 128, generator=g).bfloat16()
    v = torch.randn(blocks, bs, hkv, 128, generator=g).bfloat16()
    tables, mine = [], iter(ids)
    owned = torch.zeros(blocks, bs, dtype=torch.bool)
    for c, n in zip(ctx, need):
        row = [next(mine) for _ in range(n)]
        for b, blk in enumerate(row):
            owned[blk, :max(0, min(bs, c - b * bs))] = True
        tables.append(row + [rng.choice((-1, blocks + 5, ids[-1], 2 ** 31 - 1)) for _ in range(cols - n)])
    if poison:
        k[~owned], v[~owned] = float("nan"), float("nan")
    cu = [0]
    for n in nodes:
        cu.append(cu[-1] + n)
    total = cu[-1] + extra_rows
    fused = torch.randn(max(total, 1), (H + 2 * hkv) * 128, generator=g).bfloat16()
    q = fused[:total, :H * 128].view(total, H, 128)
    m = None
    if masks != "chain":
        words = words or max(1, -(-max(nodes + [1]) // 64))
        rows = []
        for n in nodes:
            parents = random_parents([n], rng)
            seen = []
            for j in range(n):
                bits = 1 << j
                if j:
                    bits |= seen[parents[j]]
                seen.append(bits)
            if masks == "any":
                seen = [rng.choice((0, rng.getrandbits(64 * words), rng.getrandbits(64 * words) & rng.getrandbits(64 * words))) for _ in range(n)]
            for s in seen:
                w = [(s >> (64 * x)) & (2 ** 64 - 1) for x in range(words)]
                rows.append([x - 2 ** 64 if x >> 63 else x for x in w])
        rows += [[-1] * words] * extra_rows
        m = torch.tensor(rows, dtype=torch.int64).view(total, words)
    return dict(q=q, fused=fused, k=k, v=v, cu=cu, ctx=ctx, tables=tables, masks=m, scale=128 ** -0.5, hkv=hkv, H=H, total=total)


def run_attention(c):
    q = c["fused"].to(DEV)[:c["total"], :c["H"] * 128].view(c["total"], c["H"], 128)          # a view into the projection
    return nanovllm_b200.tree_attention(q, c["k"].to(DEV), c["v"].to(DEV), i32(c["cu"]), i32(c["ctx"]), i32(c["tables"]),
                                        None if c["masks"] is None else c["masks"].to(DEV), c["scale"], c["hkv"])


def check_attention(c, out):
    want, weight = tree_attn_ref(c["q"], c["k"], c["v"], c["cu"], c["ctx"], c["tables"], c["masks"], c["scale"])
    n = c["cu"][-1]
    got, want, weight = out.double().cpu()[:n], want[:n], weight[:n]
    assert torch.isfinite(got).all()
    off = (got - want).abs() / (weight + want.abs()).clamp(min=1e-30)
    off = torch.where((weight + want.abs()) == 0, got.abs() * 1e30, off)
    assert off.max() <= BOUND, (float(off.max()), BOUND)


HEADS = [(16, 8), (32, 8), (2, 1), (5, 1), (16, 1), (24, 2), (128, 1), (3, 3)]


@pytest.mark.gpu
@pytest.mark.parametrize("H,hkv", HEADS)
@pytest.mark.parametrize("masks", ["tree", "chain", "any"])
def test_attention_heads_and_ragged_sizes(H, hkv, masks):
    ctx = [1, 2, 63, 64, 65, 127, 128, 129, 255, 256, 257, 700]
    nodes = [1, 2, 5, 64, 17, 33, 1, 64, 7, 31, 32, 63]
    c = attention_case(H, hkv, ctx, nodes, seed=H * 10 + hkv, masks=masks)
    check_attention(c, run_attention(c))
    status_ok()


@pytest.mark.gpu
@pytest.mark.parametrize("masks", ["tree", "chain", "any"])
def test_attention_large_trees_and_empty_rows(masks):
    """Trees of up to 256 nodes (more than a tile of keys, more than two of rows), sequences without nodes, without a context, and
    with more nodes than tokens; rows whose mask is empty; rows behind the last sequence."""
    ctx = [0, 300, -3, 256, 1000, 40, 64, 0, 129, 2000, 511]
    nodes = [5, 256, 3, 200, 0, 70, 64, 0, 128, 100, 255]
    c = attention_case(32, 8, ctx, nodes, seed=77, masks=masks, extra_rows=9)
    check_attention(c, run_attention(c))
    c = attention_case(4, 2, ctx, nodes, seed=78, masks=masks)
    check_attention(c, run_attention(c))
    status_ok()


@pytest.mark.gpu
@pytest.mark.parametrize("batch,ctx,nodes,H,hkv", [(1, 5000, 9, 16, 8), (1, 9001, 64, 8, 2), (2, 12345, 33, 4, 1), (3, 4097, 1, 16, 8), (40, 600, 12, 16, 8),
                                                   (1, 40000, 40, 2, 1), (170, 130, 3, 16, 8), (600, 70, 2, 2, 1), (1, 33, 8, 16, 8), (9, 1500, 64, 32, 8)])
def test_attention_long_and_many(batch, ctx, nodes, H, hkv):
    rng = random.Random(batch * ctx)
    lens = [max(nodes, ctx - rng.randint(0, ctx // 3)) for _ in range(batch)]
    c = attention_case(H, hkv, lens, [rng.randint(1, nodes) for _ in range(batch)], seed=ctx, masks=rng.choice(("tree", "any")))
    check_attention(c, run_attention(c))
    status_ok()


@pytest.mark.gpu
@pytest.mark.parametrize("H,hkv,most", [(16, 8, 8), (32, 8, 4), (5, 1, 3), (16, 1, 1), (3, 3, 16), (24, 2, 1), (28, 4, 2)])
@pytest.mark.parametrize("masks", ["tree", "chain", "any"])
def test_attention_few_nodes(H, hkv, most, masks):
    """Batches with at most 12 rows to a sequence and kv head on average: ragged contexts, none, fewer tokens than nodes, no nodes, one tile,
    and single trees of many blocks of rows between them."""
    rng = random.Random(H * most)
    ctx = [1, 2, 15, 16, 17, 63, 64, 65, 0, 127, 128, 129, 300, 700, -1, 33, 2, 1100, 64, 500] * 2
    nodes = [rng.randint(0, most) for _ in ctx]
    nodes[3], nodes[16], nodes[8] = most, most, most
    nodes[13] = 3 * most + 5
    while sum(nodes) * (H // hkv) > 12 * len(ctx):
        nodes[nodes.index(max(nodes[14:]), 14)] -= 1
    c = attention_case(H, hkv, ctx, nodes, seed=most, masks=masks, extra_rows=0)
    check_attention(c, run_attention(c))
    status_ok()


@pytest.mark.gpu
def test_attention_block_size_words_and_values():
    """Blocks of 512, masks with more words than nodes, large and small scores, an equal score everywhere."""
    for scale_q, bs, words in ((30.0, 512, 3), (1e-3, 256, 4), (0.0, 768, 1)):
        c = attention_case(16, 8, [700, 90, 1500], [20, 64, 33], seed=bs, words=words, bs=bs)
        c["fused"] = (c["fused"] * scale_q).bfloat16()
        c["q"] = c["fused"][:c["total"], :c["H"] * 128].view(c["total"], c["H"], 128)
        if scale_q < 2:
            check_attention(c, run_attention(c))
            continue
        # scores up to 30 * 7: their own error is 129 * 2^-24 * scale * sum |q||k| (about 80 * 30 * 0.088 = 211 at most 400) < 2^-8
        want, weight = tree_attn_ref(c["q"], c["k"], c["v"], c["cu"], c["ctx"], c["tables"], c["masks"], c["scale"])
        off = (run_attention(c).double().cpu() - want).abs() / (weight + want.abs()).clamp(min=1e-30)
        assert off.max() <= BOUND + 2.0 ** -8
    status_ok()


@pytest.mark.gpu
def test_attention_twice_is_the_same_and_rows_behind_stay():
    """Equal bits on every call, on another stream, and through the C entry rows outside cu_seqlens_q are left alone."""
    c = attention_case(16, 8, [4000, 1200, 300], [33, 20, 64], seed=4, extra_rows=5)
    first = run_attention(c)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        others = [run_attention(c) for _ in range(20)]
    torch.cuda.synchronize()
    n = c["cu"][-1]
    assert all(torch.equal(first[:n], o[:n]) for o in others)
    lib = _lib.load()
    q, k, v, m = c["fused"].to(DEV), c["k"].to(DEV), c["v"].to(DEV), c["masks"].to(DEV)
    cu, ctx, bt = i32(c["cu"]), i32(c["ctx"]), i32(c["tables"])
    out = torch.full((c["total"], 16, 128), 7.0, dtype=torch.bfloat16, device=DEV)
    ws = torch.full((lib.b200_tree_workspace_bytes(16, 8, 128),), 255, dtype=torch.uint8, device=DEV)      # (NaN in every float)
    _lib.check(lib.b200_tree_attn(q.data_ptr(), q.stride(0), k.data_ptr(), v.data_ptr(), k.shape[0], 256, bt.data_ptr(), bt.stride(0), bt.shape[1],
                                  cu.data_ptr(), ctx.data_ptr(), m.data_ptr(), m.shape[1], out.data_ptr(), ws.data_ptr(), ws.numel(), 3,
                                  c["total"], 16, 8, 128, c["scale"], torch.cuda.current_stream().cuda_stream))
    torch.cuda.synchronize()
    assert torch.equal(out[:n], first[:n]) and out[n:].eq(7).all()
    status_ok()


@pytest.mark.gpu
def test_attention_one_node_is_decode_and_chain_is_prefill():
    """A tree of one node is a decode step; a chain is the end of a prefill with a cached prefix.  Both sides round alike, so each
    is within the bound of the exact result, and they are within twice that of each other."""
    ctx = [5, 300, 1025, 2000]
    c = attention_case(16, 8, ctx, [1] * 4, seed=11, masks="chain")
    tree = run_attention(c)
    check_attention(c, tree)
    q = c["fused"].to(DEV)[:4, :2048].view(4, 16, 128)
    dec = nanovllm_b200.decode_attention(q, c["k"].to(DEV), c["v"].to(DEV), i32(ctx), i32(c["tables"]), c["scale"], 8)
    check_attention(c, dec.view(4, 16, 128))
    c = attention_case(16, 8, ctx, [5, 77, 64, 130], seed=12, masks="chain")
    check_attention(c, run_attention(c))
    q = c["fused"].to(DEV)[:, :2048].view(-1, 16, 128)
    cu_k = [0]
    for n in ctx:
        cu_k.append(cu_k[-1] + n)
    pre = nanovllm_b200.prefill_attention(q, c["k"].to(DEV), c["v"].to(DEV), i32(c["cu"]), i32(cu_k), 130, 2000, c["scale"], 8, i32(c["tables"]))
    check_attention(c, pre)
    status_ok()


# ---- the walk --------------------------------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("sizes,vocab,max_path", [([1], 3, 1), ([1, 2, 3, 0, 5], 2, 4), ([33, 64, 17, 0, 1, 300, 256, 257], 3, 16), ([64] * 130, 4, 40),
                                                  ([700, 5], 1, 1000), ([31, 32, 33], 2, 2)])
def test_accept_tree(sizes, vocab, max_path):
    rng = random.Random(len(sizes) * 7 + vocab)
    for chain in (False, True):
        parents = random_parents(sizes, rng, chain)
        for j in range(0, len(parents), 11):
            parents[j] = rng.choice((-1, parents[j], 5000, -9, parents[j]))         # no parent
        n = len(parents)
        draft = [rng.randrange(vocab) + (1 << 40) for _ in range(n)]
        target = [rng.randrange(vocab) + (1 << 40) for _ in range(n)]
        cu = [0]
        for s in sizes:
            cu.append(cu[-1] + s)
        cached = [rng.randrange(5000) for _ in sizes]
        ctx = [0 if rng.random() < 0.1 else c + s for c, s in zip(cached, sizes)]
        want = accept_tree_ref(draft, target, parents, cu, cached, ctx, max_path)
        cached_d = i32(cached)
        got = accept_tree(i64(draft), i64(target), i32(parents), i32(cu), cached_d, i32(ctx), max_path)
        assert [got.accepted.tolist(), got.path.tolist(), got.tokens.tolist(), got.cached_lens.tolist()] == [list(w) for w in want]
        # the lengths may be updated in place
        lib = _lib.load()
        args = [i64(draft), i64(target), i32(parents), i32(cu), cached_d, i32(ctx)]
        torch.cuda.synchronize()
        _lib.check(lib.b200_accept_tree(*[t.data_ptr() for t in args], len(sizes), n, max_path, got.accepted.data_ptr(), got.path.data_ptr(),
                                        got.tokens.data_ptr(), cached_d.data_ptr(), None))
        torch.cuda.synchronize()
        assert cached_d.tolist() == want[3]
    assert accept_tree(i64([]), i64([]), i32([]), i32([0]), i32([]), i32([]), 3).path.shape == (0, 3)
    status_ok()


# ---- the moves -------------------------------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("dtype,hkv,d,planes,bs", [(torch.bfloat16, 8, 128, (2, 3), 256), (torch.bfloat16, 1, 128, (2, 28), 256), (torch.float32, 3, 64, (5,), 16),
                                                   (torch.float16, 1, 8, (2,), 512), (torch.uint8, 1, 16, (1,), 256)])
def test_compact_bit_exact(dtype, hkv, d, planes, bs):
    """Paths whose places are sources of others, that cross blocks, do not move, run to the end; entries below their place, blocks
    outside the cache, columns outside the table."""
    rng, g = random.Random(bs + hkv), torch.Generator().manual_seed(5)
    paths = [[0, 2, 5, 6], [0, 1, 2, 3], [0, 3, 4, 60], [0, 2, 3, 4], [0], [0, 9, 10, 11], [0, 5, 1, 7], [0, 60, 61, 62], []]
    start = [bs - 3, 7, bs - 1, 0, 3, 2 * bs - 2, 20, bs, 4]
    accepted = [4, 4, 4, 3, 1, 4, 4, 9, 0]
    paths += [sorted(rng.sample(range(1, 400), 300)) for _ in range(2)]
    paths[-1] = [0] + paths[-1]
    start += [5, bs - 7]
    accepted += [300, 301]
    n = max(len(p) for p in paths)
    path = [p + [-1] * (n - len(p)) for p in paths]
    cols = -(-(max(start) + 400) // bs) + 1
    blocks = cols * len(paths) + 1
    ids = list(range(blocks))
    rng.shuffle(ids)
    tables = [ids[i * cols:(i + 1) * cols] for i in range(len(paths))]
    tables[5][2] = blocks + 3                 # a foreign id: nothing is moved there or from there
    tables[7] = [-1] * cols
    cache = torch.randint(0, 256, (*planes, blocks, bs, hkv, d * torch.empty(0, dtype=dtype).element_size()), generator=g, dtype=torch.uint8)
    dev = cache.to(DEV).view(dtype)
    flat = cache.view(-1, blocks, bs, cache.shape[-1] * hkv)
    compact_kvcache(dev, i32(path), i32(accepted), i32(start), i32(tables))
    torch.cuda.synchronize()
    compact_ref(flat, path, accepted, start, tables, bs)
    assert torch.equal(dev.view(torch.uint8).cpu(), cache)
    # a table that ends in front of the positions, a path of one column, an empty batch
    compact_kvcache(dev, i32(path), i32(accepted), i32([x + cols * bs for x in start]), i32(tables))
    compact_kvcache(dev, i32(path)[:, :1].contiguous(), i32(accepted), i32(start), i32(tables))
    compact_kvcache(dev, i32(path)[:0], i32([]), i32([]), i32(tables))
    torch.cuda.synchronize()
    assert torch.equal(dev.view(torch.uint8).cpu(), cache)
    status_ok()


# ---- together --------------------------------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("graph", [False, True])
def test_steps_together(graph):
    """Five steps of a two-layer stand-in for a model: tables, store, attention through the layer, walk, moves, blocks given
    back; eager, and captured once and replayed on changing trees.  Everything is compared with the plain restatement."""
    rng, g = random.Random(9), torch.Generator().manual_seed(9)
    H, hkv, bs, layers, cols, blocks, batch, most, words, vocab = 16, 8, 256, 2, 5, 40, 6, 40, 1, 3
    ref = BlockState([[-1] * cols for _ in range(batch)], [0] * batch, list(range(blocks)), bs)
    dev = device_state(ref, blocks)
    kv = torch.randn(2, layers, blocks, bs, hkv, 128, generator=g).bfloat16()
    kv_d = kv.to(DEV)
    att = []
    for layer in range(layers):
        a = nanovllm_b200.Attention(H, 128, 128 ** -0.5, hkv)
        a.k_cache, a.v_cache = kv_d[0, layer], kv_d[1, layer]
        att.append(a)
    from nanovllm_b200.utils.context import reset_context, set_tree_context
    cached = [250, 3, 600, 255, 90, 1000]
    dev.step(None, i32(cached), i32([0] * batch), 0)          # the prompts' blocks
    ref.step(None, cached, [0] * batch, 0)
    total = batch * most
    buf = dict(cached=i32(cached), new=i32([0] * batch), parents=i32([-1] * total), draft=i64([0] * total), target=i64([0] * total),
               qkv=torch.zeros(layers, total, (H + 2 * hkv) * 128, dtype=torch.bfloat16, device=DEV))
    result = {}

    def step():
        t = dev.step(None, buf["cached"], buf["new"], total, buf["parents"], words)
        set_tree_context(t.cu_seqlens_q, t.context_lens, t.slot_mapping, t.block_tables, t.tree_masks)
        outs = []
        for layer in range(layers):
            x = buf["qkv"][layer]
            q, k, v = x[:, :H * 128].view(total, H, 128), x[:, H * 128:(H + hkv) * 128].view(total, hkv, 128), x[:, (H + hkv) * 128:].view(total, hkv, 128)
            outs.append(att[layer](q, k, v))
        reset_context()
        a = accept_tree(buf["draft"], buf["target"], buf["parents"], t.cu_seqlens_q, buf["cached"], t.context_lens, 8)
        compact_kvcache(kv_d, a.path, a.accepted, buf["cached"], t.block_tables)
        dev.release(None, a.cached_lens)
        buf["cached"].copy_(a.cached_lens)
        result.update(t=t, outs=outs, a=a)

    captured = None
    for turn in range(5):
        new = [rng.randint(1, most) for _ in range(batch)]
        new[turn % batch] = most
        if turn == 3:
            new[1] = 0
        n = sum(new)
        parents = random_parents(new, rng) + [-1] * (total - n)
        draft, target = [[rng.randrange(vocab) for _ in range(total)] for _ in range(2)]
        x = torch.randn(layers, total, (H + 2 * hkv) * 128, generator=g).bfloat16()
        if graph and captured is None:
            # captured in front of the first step, with no nodes: nothing changes
            torch.cuda.synchronize()
            step()
            torch.cuda.synchronize()
            captured = torch.cuda.CUDAGraph()
            with torch.cuda.graph(captured):
                step()
        buf["new"].copy_(i32(new)), buf["parents"].copy_(i32(parents)), buf["draft"].copy_(i64(draft)), buf["target"].copy_(i64(target)), buf["qkv"].copy_(x)
        if graph:
            captured.replay()
        else:
            step()
        torch.cuda.synchronize()
        want = ref.step(None, cached, new, total, parents, words)
        same_step(result["t"], want, words)
        for layer in range(layers):
            k = x[layer, :, H * 128:(H + hkv) * 128].view(total, hkv, 128)
            v = x[layer, :, (H + hkv) * 128:].view(total, hkv, 128)
            for r, s in enumerate(want["slots"]):
                if s >= 0:
                    kv[0, layer, s // bs, s % bs], kv[1, layer, s // bs, s % bs] = k[r], v[r]
            c = dict(q=x[layer, :, :H * 128].view(total, H, 128), k=kv[0, layer], v=kv[1, layer], cu=want["cu_q"], ctx=want["ctx"], tables=want["tables"],
                     masks=torch.tensor(want["masks"]), scale=128 ** -0.5)
            check_attention(c, result["outs"][layer])
        accepted, path, tokens, lens = accept_tree_ref(draft, target, parents, want["cu_q"], cached, want["ctx"], 8)
        a = result["a"]
        assert [a.accepted.tolist(), a.path.tolist(), a.tokens.tolist(), a.cached_lens.tolist()] == [accepted, path, tokens, lens]
        compact_ref(kv.view(2 * layers, blocks, bs, hkv, 128), path, accepted, cached, want["tables"], bs)
        assert torch.equal(kv_d.cpu().view(torch.int16), kv.view(torch.int16))
        ref.release(None, lens)
        same_state(dev, ref)
        cached = lens
    status_ok()


@pytest.mark.gpu
def test_two_graphs_on_two_streams():
    """Two captured calls replayed at the same time, each many times: neither touches the other's scratch."""
    cases = [attention_case(16, 8, [5000, 3000], [20, 33], seed=21), attention_case(32, 8, [4000, 2500, 900], [33, 9, 64], seed=22)]
    held, graphs = [], []
    for c in cases:
        args = (c["fused"].to(DEV)[:, :c["H"] * 128].view(c["total"], c["H"], 128), c["k"].to(DEV), c["v"].to(DEV), i32(c["cu"]), i32(c["ctx"]), i32(c["tables"]),
                c["masks"].to(DEV), c["scale"], c["hkv"])
        nanovllm_b200.tree_attention(*args)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = nanovllm_b200.tree_attention(*args)
        held.append((args, out))
        graphs.append(graph)
    streams = [torch.cuda.Stream() for _ in graphs]
    for _ in range(50):
        for s, graph in zip(streams, graphs):
            with torch.cuda.stream(s):
                graph.replay()
    torch.cuda.synchronize()
    for c, (_, out) in zip(cases, held):
        check_attention(c, out)
    status_ok()


# ---- early starts ----------------------------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("H,hkv,ctx,nodes", [(16, 8, [1037], [9]), (32, 8, [700, 300, 500, 900, 40], [20, 33, 5, 64, 12]),
                                             (8, 1, [200 + 7 * i for i in range(130)], [1] * 130), (8, 4, [150 + i for i in range(60)], [12] * 60)])
def test_attention_behind_a_kernel_that_writes_its_rows(late_copy, H, hkv, ctx, nodes):
    """Rows, masks and the cache come from a kernel that lets this one start before it writes them (clusters, cut units and the
    join, few nodes)."""
    c = attention_case(H, hkv, ctx, nodes, 71, poison=False)
    late = dict(q=c["q"].contiguous(), k=c["k"], v=c["v"], masks=c["masks"])
    late = {n: t.to(DEV) for n, t in late.items()}
    cu, lens, tables = i32(c["cu"]), i32(ctx), i32(c["tables"])
    _compare(late_copy, {n: torch.zeros_like(t) for n, t in late.items()}, late, lambda: None,
             lambda m, _: (nanovllm_b200.tree_attention(m["q"], m["k"], m["v"], cu, lens, tables, m["masks"], c["scale"], hkv),))
    status_ok()


@pytest.mark.gpu
@pytest.mark.parametrize("batch,seed", [(1, 1), (40, 2), (700, 3)])
def test_tables_walk_and_moves_behind_a_kernel_that_writes_their_inputs(late_copy, batch, seed):
    rng = random.Random(seed)
    sizes = [rng.randrange(1, 20) for _ in range(batch)]
    total, cols = sum(sizes), 4
    rows = rng.sample(range(batch + 5), batch)
    cached = [rng.randrange(700) for _ in sizes]
    parents = random_parents(sizes, rng)
    cu = [0]
    for s in sizes:
        cu.append(cu[-1] + s)
    zeros = lambda late: {n: torch.zeros_like(t) for n, t in late.items()}  # noqa: E731
    fresh = lambda: DeviceBlockTables.create(batch + 5, cols, cols * batch + 3, 256, DEV)  # noqa: E731
    late = dict(rows=i32(rows), cached=i32(cached), new=i32(sizes), parents=i32(parents))

    def step(m, s):
        return (*s.step(m["rows"], m["cached"], m["new"], total, m["parents"], 1), s.tables, s.owned, s.free_blocks, s.pool)
    _compare(late_copy, zeros(late), late, fresh, step)

    def taken():
        s = fresh()
        s.step(late["rows"], late["cached"], late["new"], total)
        return s

    def release(m, s):
        s.release(m["rows"], m["keep"])
        return s.tables, s.owned, s.free_blocks, s.pool
    keep = dict(rows=late["rows"], keep=i32([rng.randrange(900) for _ in sizes]))
    _compare(late_copy, zeros(keep), keep, taken, release)
    walk = dict(draft=i64([rng.randrange(3) for _ in parents]), target=i64([rng.randrange(3) for _ in parents]), parents=late["parents"], cu=i32(cu),
                cached=late["cached"], context=i32([a + b for a, b in zip(cached, sizes)]))
    _compare(late_copy, zeros(walk), walk, lambda: None,
             lambda m, _: tuple(accept_tree(m["draft"], m["target"], m["parents"], m["cu"], m["cached"], m["context"], 6)))
    paths = [sorted(rng.sample(range(20), 6)) for _ in sizes]
    blocks = cols * batch
    cache = torch.randint(-30000, 30000, (blocks, 256, 1, 8), dtype=torch.int16, device=DEV)
    moves = dict(path=i32(paths), accepted=i32([rng.randrange(7) for _ in sizes]), start=late["cached"], tables=torch.arange(blocks, dtype=torch.int32, device=DEV).view(batch, cols))

    def compact(m, mine):
        compact_kvcache(mine, m["path"], m["accepted"], m["start"], m["tables"])
        return (mine,)
    _compare(late_copy, zeros(moves), moves, cache.clone, compact)
    status_ok()


@pytest.mark.gpu
def test_compaction_from_no_place():
    """Negative start lengths (the largest, too) move nothing."""
    cache = torch.arange(2 * 256 * 8, dtype=torch.int32, device=DEV).view(2, 256, 1, 8)
    want = cache.clone()
    compact_kvcache(cache, i32([[0, 3, 2 ** 31 - 1]] * 3), i32([3, 3, 3]), i32([-1, -2 ** 31, -3]), i32([[0], [1], [0]]))
    torch.cuda.synchronize()
    assert torch.equal(cache, want)
