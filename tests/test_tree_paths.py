"""Tree attention by the kernel that a call takes: clusters (one launch), the tcgen05 line (two: units that it cuts are joined by a
launch of their own), and the kernel for few nodes (three: the tcgen05 line behind it takes the sequences with many nodes).
Inputs, oracle and tolerance are those of test_tree_decode."""
import random

import pytest
import torch

import nanovllm_b200
from nanovllm_b200 import _lib
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
