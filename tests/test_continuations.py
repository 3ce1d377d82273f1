"""Several continuations of one prompt where caches are large, tensors lie together, weights are kept and calls are refused (ops.beams, serve.PagedCache, serve.BeamSearch)."""
import math

import pytest
import torch

from rustral_b200 import ops
from test_beams import attend64, bound

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
I32 = torch.int32


# ---- attention over a shared prefix ------------------------------------------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("dim,more", [(64, 1 << 20), (128, 1 << 21)])
def test_attention_shared_in_a_larger_cache_at_the_same_address(dim, more, cuda_status):
    """A cache of 2^19 tokens, then one at its address with `more` tokens behind them: keys and values behind the smaller one's end are read.  Weights and rounding: see `bound`."""
    n, bs, lens = 20, 16, [21 + i for i in range(20)]
    blocks = [(1 << 19) // bs, ((1 << 19) + more) // bs]
    k, v = (torch.zeros(blocks[1], bs, 1, dim, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    g = torch.Generator().manual_seed(dim)
    q = torch.randn(n, dim, generator=g).bfloat16()
    groups, shared = ops.PrefixGroups([n], "cuda"), torch.tensor([bs], dtype=I32, device="cuda")
    for count in blocks:
        pages = count - 1 - torch.randperm(1 + 2 * n, generator=g)       # the last ones
        t = torch.cat([pages[:1].expand(n, 1), pages[1:].view(n, 2)], 1).to(I32)
        held = [torch.randn(1 + 2 * n, bs, 1, dim, generator=g).bfloat16() for _ in range(2)]
        for x, h in zip((k, v), held):
            x[pages.cuda()] = h.cuda()
        got = ops.paged_attention_shared(q.cuda(), k[:count], v[:count], groups, shared, t.cuda(), torch.tensor(lens, dtype=I32, device="cuda"))
        place = torch.empty(count, dtype=torch.int64)
        place[pages] = torch.arange(len(pages))
        want, most = attend64(q, *held, place[t.long()], lens, 1.0 / math.sqrt(dim))
        assert ((got.cpu().double() - want).abs() <= bound(want, most, torch.bfloat16)).all()
