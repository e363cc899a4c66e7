"""Prefill with scales of zero and below: batches that go to the tcgen05 kernel with a positive one, dense, with the store on the
side and paged.  Probabilities and outputs are rounded to bf16 (2^-8 of each at most), the rest has 32 bits (scores as in
test_tree_decode, below 2^-11 together): |error| <= (2^-8 + 2^-11) * (sum p |v| + |out|)."""
import pytest
import torch

from workloads import cu_seqlens

DEV = "cuda:0"
BOUND = 2.0 ** -8 + 2.0 ** -11
LENS = [1, 127, 128, 129, 300, 257, 64, 500]


def exact(q, k, v, lens, scale):
    """(out, sum p |v|) of causal attention within each prompt, in 64 bits."""
    H, hkv, at, outs = q.shape[1], k.shape[1], 0, ([], [])
    for n in lens:
        x = q[at:at + n].double().view(n, hkv, H // hkv, 128)
        kk, vv = k[at:at + n].double(), v[at:at + n].double()
        s = torch.einsum("qhgd,khd->hgqk", x, kk) * scale
        p = torch.softmax(s.masked_fill(~torch.ones(n, n, dtype=torch.bool).tril(), float("-inf")), -1)
        outs[0].append(torch.einsum("hgqk,khd->qhgd", p, vv).reshape(n, H, 128))
        outs[1].append(torch.einsum("hgqk,khd->qhgd", p, vv.abs()).reshape(n, H, 128))
        at += n
    return torch.cat(outs[0]), torch.cat(outs[1])


def rows(H, hkv, seed):
    g = torch.Generator().manual_seed(seed)
    return [torch.randn(sum(LENS), h, 128, generator=g).to(torch.bfloat16) for h in (H, hkv, hkv)]


@pytest.mark.gpu
@pytest.mark.parametrize("form", ["dense", "store", "paged"])
@pytest.mark.parametrize("H,hkv", [(32, 8), (2, 1), (128, 1)])
@pytest.mark.parametrize("scale", [0.0, -128 ** -0.5])
def test_prefill_scales_that_are_not_positive(form, H, hkv, scale):
    import nanovllm_b200
    from nanovllm_b200 import _lib
    q, k, v = rows(H, hkv, H)
    cu, most = cu_seqlens(LENS).to(DEV), max(LENS)
    blocks = [-(-n // 256) for n in LENS]
    tables = torch.full((len(LENS), max(blocks)), -1, dtype=torch.int32)
    ids, slots = iter(range(sum(blocks) - 1, -1, -1)), []
    for i, n in enumerate(LENS):
        for c in range(blocks[i]):
            tables[i, c] = next(ids)
        slots += [int(tables[i, t // 256]) * 256 + t % 256 for t in range(n)]
    slots = torch.tensor(slots, dtype=torch.int32, device=DEV)
    kc, vc = (torch.zeros(sum(blocks), 256, hkv, 128, dtype=torch.bfloat16, device=DEV) for _ in range(2))
    args = (q.to(DEV), k.to(DEV), v.to(DEV))
    if form == "store":
        from nanovllm_b200.utils.context import reset_context, set_context
        att = nanovllm_b200.Attention(H, 128, scale, hkv)
        att.k_cache, att.v_cache = kc, vc
        set_context(True, cu, cu, most, most, slots)
        out = att(*args)
        reset_context()
        assert torch.equal(kc.view(-1, hkv, 128)[slots.long()], args[1]) and torch.equal(vc.view(-1, hkv, 128)[slots.long()], args[2])
    elif form == "paged":
        nanovllm_b200.store_kvcache(args[1], args[2], kc, vc, slots)
        out = nanovllm_b200.prefill_attention(args[0], kc, vc, cu, cu, most, most, scale, hkv, tables.to(DEV))
    else:
        out = nanovllm_b200.prefill_attention(*args, cu, cu, most, most, scale, hkv)
    with pytest.raises(_lib.B200AttnError, match="positive scale"):
        nanovllm_b200.prefill_attention(*args, cu, cu, most, most, scale, hkv, kernel_variant=2)
    want, weight = exact(q, k, v, LENS, scale)
    off = (out.double().cpu() - want).abs() / (weight + want.abs()).clamp(min=1e-30)
    assert off.max() <= BOUND, (float(off.max()), BOUND)
    _lib.check(_lib.load().b200_device_status())


def test_a_forced_tcgen05_prefill_is_refused_on_the_host(lib):
    call = lambda scale: lib.b200_prefill_attn(16, 2048, 16, 16, 1024, 1024, 8, None, None, 0, 0, None, 0, 0, 16, 16, 1, 8, 8, 8, 16,  # noqa: E731
                                               16, 8, 128, scale, 2, None)
    assert call(0.0) == -2 and call(-0.1) == -2 and b"positive scale" in lib.b200_last_error()
