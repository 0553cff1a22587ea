"""Run by tests/test_gpu_shared_attention.py in a process of its own with GOGGUF_B200_DEBUG=1 (the build flags are read when the
package is imported).  Attention over shared prefixes is given page tables with an id beyond the pool and a negative one, among the
shared pages and among a row's own; the debug build must record its code in the status word and read page 0 instead.  Pools and table are
views of larger buffers, so that even kernels without the check would stay inside allocated memory."""
import math
import sys

import torch

sys.path.insert(0, sys.argv[1])
from gogguf_b200.csrc import build, fast_attention as fa, tcgen05_gemm as tc   # noqa: E402

assert build.DEBUG
DEV = "cuda:0"
assert build.module("attention_shared").lib.gg_attention_shared_checked() == 1
n_pages, spare = 12, 6
status = tc.status_word(DEV)
g = torch.Generator(device=DEV).manual_seed(1)


def run(nq, nkv, d, spoil):
    k, v = (torch.randn(n_pages + spare, nkv, 64, d, device=DEV, generator=g).to(torch.bfloat16)[:n_pages] for _ in range(2))
    lists = [[0, 1, 2, 3, 4], [0, 1, 2, 5, 6], [7, 8, 9, 10, 11]]
    lens = [290, 300, 310]
    plan = fa.PrefixPlan.of_pages(lists, lens, 64, DEV)
    assert plan.groups == [(2, 3)]
    mk = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)      # noqa: E731
    table = mk(lists)
    for row, at, page in spoil:
        table[row, at] = page
    q = torch.randn(3, nq * d, device=DEV, generator=g).to(torch.bfloat16)
    out = torch.full_like(q, float("nan"))
    scratch = torch.empty(fa.shared_scratch(3, nq, nkv, d), device=DEV)
    fa.attn_decode_shared(q, k, v, out, mk([n - 1 for n in lens]), mk([0, 1, 2]), table, 64, plan, scratch, nq, nkv, d, 1 / math.sqrt(d), together=True)
    code = int(status.item())
    status.zero_()
    assert torch.isfinite(out).all()
    return code


for nq, nkv, d in ((8, 2, 128), (16, 1, 64), (6, 2, 72)):
    assert run(nq, nkv, d, []) == 0
    for spoil in ([(0, 1, n_pages + 2)], [(0, 2, -1)], [(1, 3, n_pages)], [(2, 4, -7)], [(0, 0, -1), (1, 0, -1)]):
        assert run(nq, nkv, d, spoil) == 54, (nq, nkv, d, spoil)
print("debug shared ok")
