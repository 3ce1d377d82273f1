"""Child process of tests/test_continuations.py: runs with RUSTRAL_BOUNDS=1, i.e. on the index-checking build of the kernel library, and feeds attention over a
shared prefix tables that name blocks which are not there (the kernels read block 0 in their place in every build; this build also says so)."""
import json

import torch

from rustral_b200 import _native as N
from rustral_b200 import ops

lib = N.kernels()
assert N.KERNEL_LIB == "librb200_kernels_bounds.so" and lib.rb_build_flags() & 1, "not the checking build"
lib.rb_init()
N.read_status(clear=True)
out, dev, bs, blocks = {}, "cuda", 16, 80
g = torch.Generator().manual_seed(0)
k, v = (torch.randn(blocks, bs, 2, 64, generator=g).bfloat16().to(dev) for _ in range(2))
for name, n in (("few", 4), ("many", 24)):
    q = torch.randn(n, 256, generator=g).bfloat16().to(dev)
    table = torch.tensor([[1, 2, 3 + i] for i in range(n)], dtype=torch.int32)
    lens, shared = torch.tensor([33 + i % 15 for i in range(n)], dtype=torch.int32, device=dev), torch.tensor([32], dtype=torch.int32, device=dev)
    groups = ops.PrefixGroups([n], dev)
    for kind, at in (("ok", None), ("shared", (0, 1)), ("own", (2, 2))):
        for bad in (-1, -1 << 31, blocks, (1 << 31) - 1) if at else (3,):
            t = table.clone()
            if at:
                t[at] = bad
            got = ops.paged_attention_shared(q, k, v, groups, shared, t.to(dev), lens)
            torch.cuda.synchronize()
            bits, where = N.read_status(clear=True)
            t[(t < 0) | (t >= blocks)] = 0
            same = torch.equal(got, ops.paged_attention_shared(q, k, v, groups, shared, t.to(dev), lens))
            out.setdefault(f"{name}_{kind}", []).append([int(bits), int(where), same])
print(json.dumps(out))
