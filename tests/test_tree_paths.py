"""Tree attention by the kernel that a call takes: clusters (one launch), the tcgen05 line (two: units that it cuts are joined by a
launch of their own), and the kernel for few nodes (three: the tcgen05 line behind it takes the sequences with many nodes).
Inputs, oracle and tolerance are those of test_tree_decode."""
import random
from types import SimpleNamespace

import pytest
import torch

import nanovllm_b200
from nanovllm_b200 import _lib
from test_early_start import _compare, late_copy  # noqa: F401  (late_copy is a fixture)
from test_tree_decode import DEV, attention_case, check_attention, i32, status_ok

CLUSTER, LINE, FEW = "cluster", "line", "few"


def widened(c, cols):
    """The same case with `cols` columns of stale ids behind its tables: the host's rule goes by their width."""
    return dict(c, tables=[row + [2 ** 31 - 1] * (cols - len(row)) for row in c["tables"]])


def on_device(c):
    q = c["fused"].to(DEV)[:c["total"], :c["H"] * 128].view(c["total"], c["H"], 128)
    return (q, c["k"].to(DEV), c["v"].to(DEV), i32(c["cu"]), i32(c["ctx"]), i32(c["tables"]),
            None if c["masks"] is None else c["masks"].to(DEV), c["scale"], c["hkv"])


def run_on(path, args):
    """The call's result, and a look whether it took that kernel."""
    before = _lib.load().b200_launch_count()
    out = nanovllm_b200.tree_attention(*args)
    assert _lib.load().b200_launch_count() - before == {CLUSTER: 1, LINE: 2, FEW: 3}[path]
    return out


def case_on(path, seed, masks="tree", H=16, hkv=8):
    """Ragged contexts and trees that the host's rule sends to that kernel (16/8 heads)."""
    rng = random.Random(seed)
    ctx = [1, 300, 64, 700, 129, 40, 257, 90, 512, 33, 128, 65]
    if path == CLUSTER:
        return attention_case(H, hkv, ctx[:2], [1, 30], seed, masks=masks)
    if path == FEW:
        return attention_case(H, hkv, ctx, [rng.randint(1, 8) for _ in ctx[:-4]] + [1, 2, 0, 3], seed, masks=masks)
    return attention_case(H, hkv, ctx, [rng.randint(1, 90) for _ in ctx], seed, masks=masks)


# ---- scales ----------------------------------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("path", [CLUSTER, LINE, FEW])
@pytest.mark.parametrize("scale", [0.0, -0.0, -128 ** -0.5, 2.0 ** -140, -2.0 ** -149])
@pytest.mark.parametrize("masks", ["any", "chain"])
def test_attention_scales_that_are_not_positive(path, scale, masks):
    """Of scale 0 the mean of what a row sees, of a negative one the softmax of turned scores (errors are those of the same
    scale without its sign); tiny ones are a mean, too."""
    c = dict(case_on(path, 31, masks), scale=scale)
    check_attention(c, run_on(path, on_device(c)))
    status_ok()


# ---- how much one call may have ----------------------------------------------------------------------------------
@pytest.mark.gpu
def test_attention_under_wide_tables():
    """The limit on a call is of the kernel that it takes: its own blocks of nodes and key tiles, not the other's.  Beyond the limit of the kernel
    for few nodes the tcgen05 kernel runs, beyond that one's the call is refused."""
    rng = random.Random(3)
    c = attention_case(32, 8, [rng.randint(20, 300) for _ in range(40)], [20] * 40, 41)
    narrow = run_on(LINE, on_device(c))
    check_attention(c, narrow)
    args = list(on_device(c))
    wide = torch.full((40, 40000), 2 ** 31 - 1, dtype=torch.int32, device=DEV)
    wide[:, :args[5].shape[1]] = args[5]
    args[5] = wide
    assert torch.equal(run_on(LINE, args), narrow)
    c = attention_case(16, 8, [rng.randint(1, 300) for _ in range(100)], [1] * 100, 42)
    args = list(on_device(c))
    wide = torch.full((100, 150000), -1, dtype=torch.int32, device=DEV)
    wide[:, :args[5].shape[1]] = args[5]
    args[5] = wide
    check_attention(c, run_on(LINE, args))
    empty = torch.zeros(1001, dtype=torch.int32, device=DEV)
    args[0], args[3], args[4] = torch.zeros(1000, 16, 128, dtype=torch.bfloat16, device=DEV), empty, empty[:1000]
    args[5], args[6] = torch.full((1000, 20000), -1, dtype=torch.int32, device=DEV), torch.zeros(1000, 1, dtype=torch.int64, device=DEV)
    with pytest.raises(_lib.B200AttnError, match="too many for one call"):
        nanovllm_b200.tree_attention(*args)
    status_ok()


# ---- batches with few nodes to most sequences -----------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("H,hkv,limit", [(16, 8, 16), (32, 8, 8), (5, 1, 6), (16, 1, 2), (3, 3, 32), (28, 4, 4)])
@pytest.mark.parametrize("masks", ["tree", "chain", "any"])
def test_attention_large_trees_among_small_ones(H, hkv, limit, masks):
    """Sequences with more than `limit` nodes (twice what a unit of 16 rows holds) go to the other kernel, those with as many do not: each
    reads its keys a few times, whatever the mean.  Among both kinds some have no context or fewer tokens than nodes."""
    rng = random.Random(limit)
    ctx = [1, 300, 65, 700, 0, 257, 40, -1, 512, 33, 128, 64]
    nodes = [1, limit, limit + 1, 256, limit + 3, limit, 2, 1, 2 * limit + 1, limit + 1, 1, 0]
    while sum(nodes) * (H // hkv) > 12 * len(ctx) or len(ctx) * hkv <= 74:
        ctx.append(rng.choice((1, 16, 90, 200)))
        nodes.append(rng.choice((0, 1)))
    c = attention_case(H, hkv, ctx, nodes, seed=H, masks=masks, extra_rows=1)
    c["total"] -= 1                                     # (rows behind the last sequence would count in the mean)
    c["q"], c["masks"] = c["q"][:-1], c["masks"] if c["masks"] is None else c["masks"][:-1]
    out = run_on(FEW, on_device(c))
    check_attention(c, out)
    assert all(torch.equal(out, run_on(FEW, on_device(c))) for _ in range(3))
    status_ok()


@pytest.mark.gpu
def test_attention_large_trees_alone_and_long():
    """One tree on a long context among sequences without nodes (padded rows of a graph) and with one; no sequence can have many."""
    c = attention_case(16, 8, [9000] + [0] * 20 + [200] * 40, [60] + [0] * 20 + [1] * 40, 51)
    check_attention(c, run_on(FEW, on_device(c)))
    c = attention_case(16, 8, [9000] + [3] * 49, [250] + [0] * 49, 52)
    check_attention(c, run_on(FEW, on_device(c)))
    c = attention_case(16, 8, [300] * 12, [1] * 12, 53)            # (12 nodes in all: two launches)
    check_attention(c, run_on(LINE, on_device(c)))
    status_ok()


# ---- scratch, and the same bits ---------------------------------------------------------------------------------
def cut_case(path, seed):
    """Contexts so long that the line cuts units (and, of few nodes, two trees that the tcgen05 kernel gets)."""
    rng = random.Random(seed)
    if path == LINE:
        return attention_case(32, 8, [rng.randint(200, 3000) for _ in range(11)], [rng.randint(9, 64) for _ in range(11)], seed, extra_rows=3)
    return attention_case(16, 8, [rng.randint(100, 2500) for _ in range(30)] + [3500, 2900], [rng.randint(1, 4) for _ in range(30)] + [40, 33], seed, extra_rows=3)


def through_c(c, args, ws):
    """The same call through the C entry, with this workspace and an output of sevens."""
    lib, out = _lib.load(), torch.full((c["total"], c["H"], 128), 7.0, dtype=torch.bfloat16, device=DEV)
    q, k, v, cu, ctx, bt, m, scale, hkv = args
    _lib.check(lib.b200_tree_attn(q.data_ptr(), q.stride(0), k.data_ptr(), v.data_ptr(), k.shape[0], 256, bt.data_ptr(), bt.stride(0), bt.shape[1], cu.data_ptr(),
                                  ctx.data_ptr(), m.data_ptr(), m.shape[1], out.data_ptr(), ws.data_ptr(), ws.numel(), len(ctx), c["total"], c["H"], hkv, 128, scale,
                                  torch.cuda.current_stream().cuda_stream))
    return out


@pytest.mark.gpu
@pytest.mark.parametrize("path", [LINE, FEW])
def test_cut_units_give_the_same_bits_whatever_the_workspace_held(path):
    """20 calls on another stream, workspaces of NaN, of zeros and of another call's results; rows behind the last sequence stay."""
    c, other = cut_case(path, 61), cut_case(LINE if path == FEW else FEW, 62)
    args, others = on_device(c), on_device(other)
    n = c["cu"][-1]
    first = run_on(path, args)
    check_attention(c, first)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = [run_on(path, args) for _ in range(20)]
    torch.cuda.synchronize()
    assert all(torch.equal(first[:n], o[:n]) for o in again)
    size = max(_lib.load().b200_tree_workspace_bytes(x["H"], x["hkv"], 128) for x in (c, other))
    ws = torch.full((size,), 255, dtype=torch.uint8, device=DEV)
    outs = [through_c(c, args, ws)]
    ws.zero_()
    outs.append(through_c(c, args, ws))
    through_c(other, others, ws)
    outs.append(through_c(c, args, ws))
    torch.cuda.synchronize()
    for out in outs:
        assert torch.equal(out[:n], first[:n]) and out[n:].eq(7).all()
    status_ok()


@pytest.mark.gpu
@pytest.mark.parametrize("paths", [(LINE, LINE), (LINE, FEW), (FEW, FEW)])
def test_two_graphs_that_cut_units_on_two_streams(paths):
    """Replayed at the same time, many times, they give what the calls give one behind the other: the scratch is each one's own."""
    held, graphs = [], []
    for i, path in enumerate(paths):
        c = cut_case(path, 65 + i)
        args = on_device(c)
        alone = run_on(path, args)
        check_attention(c, alone)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = run_on(path, args)
        held.append((args, out, alone, c["cu"][-1]))
        graphs.append(graph)
    streams = [torch.cuda.Stream() for _ in graphs]
    for _ in range(10):
        for _ in range(10):
            for s, graph in zip(streams, graphs):
                with torch.cuda.stream(s):
                    graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(out[:n], alone[:n]) for _, out, alone, n in held)
    status_ok()


# ---- many sequences -----------------------------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("path,batch", [(LINE, 513), (LINE, 1100), (FEW, 700)])
def test_attention_of_more_sequences_than_a_block_has_threads(path, batch):
    """The line's sum takes two passes over the lengths; of few nodes some sequences are the other kernel's."""
    rng = random.Random(batch)
    ctx = [rng.choice((1, 20, 64, 130, 200)) for _ in range(batch)]
    nodes = [rng.randint(5, 9) if path == LINE else rng.choice((0, 1, 1, 2)) for _ in range(batch)]
    if path == FEW:
        nodes[3], nodes[600], nodes[699], ctx[600] = 40, 64, 35, 1500
    c = attention_case(2, 1, ctx, nodes, batch)
    check_attention(c, run_on(path, on_device(c)))
    status_ok()


# ---- behind the step's tables and the fused producer ----------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("cols", [5, 160])
def test_tables_of_a_step_then_the_layer_behind_the_fused_producer(cols):
    """A tree step as a model's layer runs it with QK-norm, rotary embedding and store in one kernel: positions by depth and slots from
    DeviceBlockTables.step, attention on its tables of 5 and of 160 columns, whose spare ones hold -1."""
    from nanovllm_b200.engine.block_tables import DeviceBlockTables
    from nanovllm_b200.layers.qk_norm_rope import fused_attention_forward, qk_norm_rope_store
    from nanovllm_b200.utils.context import reset_context, set_tree_context
    from oracle.qk_norm_rope_oracle import qk_norm_rope_ref, rope_cos_sin_cache
    from oracle.tree_oracle import BlockState
    from test_qk_norm_rope import _one_step
    from test_tree_decode import random_parents, same_step
    rng, g = random.Random(cols), torch.Generator().manual_seed(cols)
    H, hkv, blocks, cached, new = 16, 8, 30, [250, 3, 600, 1000], [17, 1, 40, 9]
    total = sum(new) + 2                                                    # two rows behind the last sequence
    ref, dev = BlockState([[-1] * cols for _ in new], [0] * 4, list(range(blocks - 1, -1, -1)), 256), DeviceBlockTables.create(4, cols, blocks, 256, DEV)
    parents = random_parents(new, rng) + [-1, -1]
    dev.step(None, i32(cached), i32([0] * 4), 0), ref.step(None, cached, [0] * 4, 0)
    t, want = dev.step(None, i32(cached), i32(new), total, i32(parents), 1), ref.step(None, cached, new, total, parents, 1)
    same_step(t, want, 1)
    kv = torch.randn(2, blocks, 256, hkv, 128, generator=g).bfloat16().to(DEV)
    att = nanovllm_b200.Attention(H, 128, 128 ** -0.5, hkv)
    att.k_cache, att.v_cache = kv[0], kv[1]
    qkv = torch.randn(total, (H + 2 * hkv) * 128, generator=g).bfloat16()
    weights = [(1.0 + 0.1 * torch.randn(128, generator=g)).bfloat16() for _ in range(2)]
    table = rope_cos_sin_cache(128, 2048, 1e6)
    norm = lambda w: SimpleNamespace(weight=w.to(DEV), eps=1e-6)  # noqa: E731
    layer = SimpleNamespace(qkv_proj=lambda x: x, o_proj=lambda x: x, attn=att, q_norm=norm(weights[0]), k_norm=norm(weights[1]),
                            rotary_emb=SimpleNamespace(cos_sin_cache=table.to(DEV)), num_heads=H, num_kv_heads=hkv)
    set_tree_context(t.cu_seqlens_q, t.context_lens, t.slot_mapping, t.block_tables, t.tree_masks)
    before = _lib.load().b200_launch_count()
    out = fused_attention_forward(layer, t.positions, qkv.to(DEV)).view(total, H, 128)
    assert _lib.load().b200_launch_count() - before == (2 if cols == 5 else 3)      # the producer, and a cluster or the line with its join
    reset_context()
    q, k, v = qk_norm_rope_ref(qkv, torch.tensor(want["positions"]), *weights, table, 1e-6, H, hkv, 128)
    q_dev, k_dev, _ = qk_norm_rope_store(qkv.to(DEV), t.positions, weights[0].to(DEV), weights[1].to(DEV), table.to(DEV), 1e-6, H, hkv)
    n = sum(new)
    _one_step(q_dev[:n].cpu(), q[:n]), _one_step(k_dev[:n].cpu(), k[:n])
    cache = kv.cpu()
    for r, s in enumerate(want["slots"][:n]):
        assert torch.equal(cache[0, s // 256, s % 256], k_dev[r].cpu()) and torch.equal(cache[1, s // 256, s % 256], v[r])
    check_attention(dict(q=q_dev.cpu(), k=cache[0], v=cache[1], cu=want["cu_q"], ctx=want["ctx"], tables=want["tables"], masks=torch.tensor(want["masks"]),
                         scale=128 ** -0.5), out)
    status_ok()


@pytest.mark.gpu
@pytest.mark.parametrize("path", [LINE, FEW])
def test_cut_units_behind_a_kernel_that_writes_its_rows(late_copy, path):
    """Rows, masks and the cache come from a kernel that lets this one start before it writes them; of few nodes two launches stand between
    that kernel and the one that takes the large trees."""
    c = cut_case(path, 81)
    late = {x: c[x].contiguous().to(DEV) for x in ("q", "k", "v", "masks")}
    for x in "kv":
        late[x] = torch.nan_to_num(late[x])
    cu, lens, tables, n = i32(c["cu"]), i32(c["ctx"]), i32(c["tables"]), c["cu"][-1]
    _compare(late_copy, {x: torch.zeros_like(t) for x, t in late.items()}, late, lambda: None,
             lambda m, _: (nanovllm_b200.tree_attention(m["q"], m["k"], m["v"], cu, lens, tables, m["masks"], c["scale"], c["hkv"])[:n],))
    status_ok()
