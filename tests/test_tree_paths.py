"""Tree attention by the kernel that a call takes: clusters (one launch), the tcgen05 line and the kernel for few nodes (more:
units that the line cuts are joined by a launch of their own).  Inputs, oracle and tolerance are those of test_tree_decode."""
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
    """The call's result, and a look whether it took that kernel: a cluster is one launch, the others come with a join."""
    before = _lib.load().b200_launch_count()
    out = nanovllm_b200.tree_attention(*args)
    assert (_lib.load().b200_launch_count() - before == 1) == (path == CLUSTER)
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
