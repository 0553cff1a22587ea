"""Decode attention over prefixes that rows share (csrc/attention_shared.cu) against the formula in 64 bits.

Tolerance.  The kernels round the weights p_j to bfloat16 before they meet the values (half a step: 2^-8 of each, so at most
2^-8 of A = sum p_j |v_j| / sum p_j), and the result once more (2^-8 of it).  Scores and sums are 32-bit: a score's error is
at most d 2^-24 scale sum |q_i k_i|, below 2e-4 for the numbers here, and weighs twice (numerator and denominator); a tenth
of 2^-8 A covers it."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

PAGE = 64


def layout(groups, prefix, own, seed):
    """groups: rows per prefix; prefix: pages per prefix; own: (least, most) positions of a row's own.  Page lists, lengths."""
    g = torch.Generator().manual_seed(seed)
    lists, lengths, need = [], [], 0
    for n, pages in zip(groups, prefix):
        shared = list(range(need, need + pages))
        need += pages
        for _ in range(n):
            tokens = int(torch.randint(own[0], own[1] + 1, (1,), generator=g))
            mine = -(-tokens // PAGE)
            lists.append(shared + list(range(need, need + mine)))
            need += mine
            lengths.append(pages * PAGE + tokens)
    ids = torch.randperm(need + 3, generator=g)
    order = torch.randperm(len(lists), generator=g).tolist()
    return [ids[torch.tensor(lists[r])].tolist() for r in order], [lengths[r] for r in order], need + 3


def reference(q, k, v, lists, lengths, nq, nkv, scale, sink=None, gate=None, out_scale=1.0):
    d, dv, G = k.shape[-1], v.shape[-1], nq // nkv
    out = torch.empty(len(lists), nq * dv, dtype=torch.float64, device=q.device)
    size = torch.empty_like(out)
    for r, pages in enumerate(lists):
        at = torch.tensor(pages, device=q.device)
        keys = k[at].double().transpose(1, 2).reshape(-1, nkv, d)[:lengths[r]].repeat_interleave(G, 1)
        vals = v[at].double().transpose(1, 2).reshape(-1, nkv, dv)[:lengths[r]].repeat_interleave(G, 1)
        s = torch.einsum("nhd,hd->hn", keys, q[r].double().view(nq, d)) * scale
        if sink is not None:
            p = torch.softmax(torch.cat([s, sink.double()[:, None]], 1), 1)[:, :-1]
        else:
            p = torch.softmax(s, 1)
        f = out_scale * (torch.sigmoid(gate[r, :nq * dv].double()) if gate is not None else 1.0)
        out[r] = torch.einsum("hn,nhd->hd", p, vals).reshape(-1) * f
        size[r] = torch.einsum("hn,nhd->hd", p, vals.abs()).reshape(-1) * f
    return out, size


def check(got, out, size):
    tol = 2.0 ** -8 * (1.1 * size + out.abs()) + 1e-30
    err = (got.double() - out).abs()
    assert torch.isfinite(got).all()
    assert (err <= tol).all(), f"worst {float((err / tol).max())}"


class Setup:
    def __init__(self, groups, prefix, own, nq, nkv, d, dv=None, sink=False, gate=False, seed=0, size=1.5):
        dv = dv or d
        dev = torch.device("cuda")
        self.nq, self.nkv, self.d, self.dv, self.scale = nq, nkv, d, dv, 1.0 / math.sqrt(d)
        self.lists, self.lengths, pages = layout(groups, prefix, own, seed)
        g = torch.Generator(device=dev).manual_seed(seed)
        self.k = torch.randn(pages, nkv, PAGE, d, generator=g, device=dev).to(torch.bfloat16)
        self.v = torch.randn(pages, nkv, PAGE, dv, generator=g, device=dev).to(torch.bfloat16)
        T = self.T = len(self.lists)
        self.q = (torch.randn(T, nq * d, generator=g, device=dev) * size).to(torch.bfloat16)
        self.sink = torch.randn(nq, generator=g, device=dev) if sink else None
        self.gate = torch.randn(T, nq * dv + 8, generator=g, device=dev).to(torch.bfloat16) if gate else None
        width = max(map(len, self.lists)) + 2
        self.table = torch.tensor([p + [0] * (width - len(p)) for p in self.lists], dtype=torch.int32, device=dev)
        self.positions = torch.tensor([n - 1 for n in self.lengths], dtype=torch.int32, device=dev)
        self.rows = torch.arange(T, dtype=torch.int32, device=dev)
        self.out = torch.full((T + 2, nq * dv), 7.0, dtype=torch.bfloat16, device=dev)

    def run(self, plan=None, scratch=None, **kw):
        from gogguf_b200.csrc import fast_attention as A
        if plan is None:
            plan = A.PrefixPlan.of_pages(self.lists, self.lengths, PAGE, "cuda")
        if scratch is None:
            scratch = torch.full((A.shared_scratch(self.T, self.nq, self.nkv, self.dv, kw.get("shares")),), math.nan, device="cuda")
        kw = {"sink": self.sink, "gate": self.gate, "dv": self.dv, "together": True, **kw}
        A.attn_decode_shared(self.q, self.k, self.v, self.out, self.positions, self.rows, self.table, PAGE, plan, scratch, self.nq,
                             self.nkv, self.d, self.scale, **kw)
        from gogguf_b200.csrc.tcgen05_gemm import check_status
        check_status(self.q.device)
        return self.out[:self.T]

    def want(self, **kw):
        return reference(self.q, self.k, self.v, self.lists, self.lengths, self.nq, self.nkv, self.scale, self.sink, self.gate, **kw)


CASES = {
    "two rows, a page": dict(groups=[2], prefix=[1], own=(1, 1), nq=2, nkv=2, d=64),
    "eight rows of 128": dict(groups=[8], prefix=[9], own=(1, 200), nq=32, nkv=8, d=128),
    "more rows than a tile": dict(groups=[45], prefix=[5], own=(60, 70), nq=8, nkv=2, d=64),
    "tiles of unequal size": dict(groups=[9], prefix=[13], own=(64, 64), nq=32, nkv=2, d=128),
    "one kv head, many parts": dict(groups=[3], prefix=[700], own=(1, 5), nq=4, nkv=1, d=64),
    "prefixes of several lengths and rows alone": dict(groups=[4, 1, 7, 2, 1], prefix=[6, 4, 31, 1, 2], own=(1, 130), nq=12, nkv=4, d=128),
    "forty groups": dict(groups=[2] * 40, prefix=[1 + i % 4 for i in range(40)], own=(1, 9), nq=4, nkv=2, d=64),
    "odd head sizes": dict(groups=[6, 3], prefix=[7, 3], own=(1, 100), nq=15, nkv=5, d=72, dv=40, sink=True),
    "values wider than keys": dict(groups=[5], prefix=[11], own=(1, 70), nq=6, nkv=2, d=40, dv=120),
    "keys wider than values": dict(groups=[5], prefix=[11], own=(1, 70), nq=6, nkv=2, d=128, dv=64, gate=True),
    "sinks and gates": dict(groups=[8, 2], prefix=[12, 20], own=(30, 300), nq=16, nkv=4, d=128, sink=True, gate=True),
    "twelve heads, values wider": dict(groups=[5, 1], prefix=[11, 3], own=(1, 200), nq=24, nkv=2, d=40, dv=120, sink=True),
    "eleven heads, keys wider": dict(groups=[4], prefix=[3], own=(1, 200), nq=11, nkv=1, d=128, dv=64),
    "ten heads of 64": dict(groups=[7], prefix=[5], own=(1, 300), nq=20, nkv=2, d=64, gate=True),
    "sixteen small heads": dict(groups=[9, 2], prefix=[4, 20], own=(1, 90), nq=16, nkv=1, d=32, dv=24),
    "nine heads of 80 and 72": dict(groups=[3, 1], prefix=[9, 9], own=(60, 140), nq=36, nkv=4, d=80, dv=72, sink=True),
    "eight small heads": dict(groups=[9, 2], prefix=[4, 20], own=(1, 90), nq=16, nkv=2, d=24, dv=56),
    "eight heads of 128, sixteen wide scores": dict(groups=[3], prefix=[8], own=(1, 200), nq=8, nkv=1, d=128, size=60.0),
    "scores far apart": dict(groups=[6], prefix=[10], own=(1, 90), nq=8, nkv=4, d=64, size=60.0),
}


@pytest.mark.parametrize("case", CASES)
def test_matches_the_formula(case):
    s = Setup(**CASES[case], seed=len(case))
    got = s.run()
    if case == "scores far apart":
        # (scores of up to some 2,000: their own 32-bit errors, 64 2^-24 of sum |q k| scale, reach 1e-2)
        out, size = s.want()
        assert ((got.double() - out).abs() <= 2.0 ** -8 * (1.1 * size + out.abs()) + 4e-2 * size).all()
        return
    check(got, *s.want())
    assert (s.out[s.T:] == 7.0).all()                   # rows behind the last one stay as they were


@pytest.mark.parametrize("kw", [dict(groups=[3, 2], prefix=[4, 9], own=(1, 700), nq=32, nkv=4, d=128),
                                dict(groups=[4], prefix=[3], own=(1, 300), nq=32, nkv=2, d=128),
                                dict(groups=[70, 1, 1], prefix=[2, 30, 1], own=(1, 300), nq=24, nkv=8, d=128),
                                dict(groups=[300], prefix=[1], own=(1, 4), nq=4, nkv=4, d=64)])
def test_own_pages_and_a_factor(kw):
    s = Setup(**kw)
    for runs, shares in ((None, None), (1, 1), (3, 3), (296, 8)):
        check(s.run(out_scale=0.5, runs=runs, shares=shares), *s.want(out_scale=0.5))


def test_rows_that_share_nothing():
    from gogguf_b200.csrc import fast_attention as A
    s = Setup(groups=[1] * 37, prefix=[1 + i % 5 for i in range(37)], own=(1, 90), nq=8, nkv=2, d=128)
    check(s.run(plan=A.PrefixPlan([], 37, "cuda")), *s.want())


@pytest.mark.parametrize("kw", [dict(groups=[3, 1], prefix=[2, 4], own=(1, 100), nq=8, nkv=2, d=72, dv=40), dict(groups=[2], prefix=[90], own=(1, 9), nq=4, nkv=2, d=64)])
def test_apart_where_that_is_quicker(kw):
    from gogguf_b200.csrc import fast_attention as A
    s = Setup(**kw)
    pays = A.prefix_pays([(n, p) for n, p in zip(kw["groups"], kw["prefix"]) if n > 1], s.T, s.nkv)
    for together in (None, False, True):
        check(s.run(together=together), *s.want())
    got = s.run(together=None).clone()
    assert torch.equal(got, s.run(together=pays))


def test_padding_rows_and_two_tokens_of_a_sequence():
    """A padded batch (rows without a sequence), and two tokens of one sequence as two members of a group."""
    from gogguf_b200.csrc import fast_attention as A
    s = Setup(groups=[3], prefix=[4], own=(5, 50), nq=8, nkv=2, d=64)
    s.lists, s.lengths = s.lists[:2] + [s.lists[0]], [s.lengths[0], s.lengths[1], s.lengths[0] - 2]
    s.rows = torch.tensor([0, 1, 0], dtype=torch.int32, device="cuda")
    s.positions = torch.tensor([n - 1 for n in s.lengths], dtype=torch.int32, device="cuda")
    want = s.want()
    check(s.run(plan=A.PrefixPlan([([2, 0, 1], 4)], 3, "cuda")), *want)
    s.rows = torch.tensor([0, -1, 0], dtype=torch.int32, device="cuda")
    got = s.run(plan=A.PrefixPlan([([2, 0], 4)], 3, "cuda"))
    check(got[[0, 2]], want[0][[0, 2]], want[1][[0, 2]])
    assert (got[1] == 0).all()                          # as the unshared kernel leaves padding
    got = s.run(plan=A.PrefixPlan([([1, 2, 0], 4)], 3, "cuda"))
    check(got[[0, 2]], want[0][[0, 2]], want[1][[0, 2]])      # a group whose first row is padding
    assert (got[1] == 0).all()


def test_a_plan_longer_than_the_table():
    """Refused where the plan's pages are known; packed words that say so read no further than the table, and other rows are right."""
    from gogguf_b200.csrc import fast_attention as A
    from gogguf_b200.csrc.build import KernelError
    s = Setup(groups=[2, 3], prefix=[4, 6], own=(5, 50), nq=8, nkv=2, d=64)
    groups = [([0, 1], 9000), ([2, 3, 4], s.table.shape[1] + 1)]
    with pytest.raises(KernelError, match="longer than the table"):
        s.run(plan=A.PrefixPlan(groups, s.T, "cuda"))
    words = A.PrefixPlan([([r for r in range(s.T) if s.lists[r][0] == s.lists[0][0]], 9000)], s.T, "cuda").words
    other = [r for r in range(s.T) if s.lists[r][0] != s.lists[0][0]]
    got = s.run(plan=A.PrefixPlan.over(words, s.T))
    check(got[other], *(w[other] for w in s.want()))


def test_calls_one_after_the_other_in_one_scratch():
    """Six calls behind each other, of two steps in turn, in the same scratch, launched one by one and captured."""
    from gogguf_b200.csrc import fast_attention as A
    steps = [Setup(groups=[5, 3], prefix=[8, 40], own=(1, 100), nq=8, nkv=2, d=128, seed=1), Setup(groups=[7, 1], prefix=[19, 2], own=(1, 300), nq=8, nkv=2, d=128, seed=2)]
    plans = [A.PrefixPlan.of_pages(s.lists, s.lengths, PAGE, "cuda") for s in steps]
    scratch = torch.empty(A.shared_scratch(8, 8, 2, 128), device="cuda")
    outs = [torch.full_like(steps[0].out, 7.0) for _ in range(6)]

    def calls():
        for i, out in enumerate(outs):
            s = steps[i % 2]
            A.attn_decode_shared(s.q, s.k, s.v, out, s.positions, s.rows, s.table, PAGE, plans[i % 2], scratch, 8, 2, 128, s.scale, together=True)

    calls()
    torch.cuda.synchronize()
    first = [o.clone() for o in outs]
    for i, out in enumerate(first):
        check(out[:8], *steps[i % 2].want())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        calls()
    for out in outs:
        out.fill_(5.0)
    for _ in range(3):
        graph.replay()
    torch.cuda.synchronize()
    for out, was in zip(outs, first):
        assert torch.equal(out[:8], was[:8])


def test_captured_with_plans_that_change():
    """A captured launch follows the plan's words, which a step rewrites."""
    from gogguf_b200.csrc import fast_attention as A
    s = Setup(groups=[5, 3], prefix=[8, 12], own=(1, 100), nq=8, nkv=2, d=128)
    want = s.want()
    full = A.PrefixPlan.of_pages(s.lists, s.lengths, PAGE, "cuda")
    words = torch.empty_like(full.words)
    plan = A.PrefixPlan.over(words, s.T)
    scratch = torch.empty(A.shared_scratch(s.T, 8, 2, 128), device="cuda")
    words.copy_(full.words)
    s.run(plan=plan, scratch=scratch)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        A.attn_decode_shared(s.q, s.k, s.v, s.out, s.positions, s.rows, s.table, PAGE, plan, scratch, 8, 2, 128, s.scale, together=True)
    members = [r for r in range(s.T) if s.lists[r][0] == s.lists[0][0]]
    for other in (full, A.PrefixPlan([], s.T, "cuda"), A.PrefixPlan([(members, 3)], s.T, "cuda"), full):
        words.copy_(other.words)
        s.out.fill_(3.0)
        graph.replay()
        check(s.out[:s.T], *want)


def test_two_streams_with_scratch_of_their_own():
    a = Setup(groups=[6], prefix=[40], own=(1, 100), nq=8, nkv=2, d=128, seed=1)
    b = Setup(groups=[3, 9], prefix=[30, 5], own=(1, 100), nq=8, nkv=2, d=128, seed=2)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(5):
        for s, stream in zip((a, b), streams):
            with torch.cuda.stream(stream):
                s.run()
    torch.cuda.synchronize()
    for s in (a, b):
        check(s.out[:s.T], *s.want())


def test_the_same_bits_every_time():
    s = Setup(groups=[11], prefix=[70], own=(1, 300), nq=16, nkv=4, d=128)
    first = s.run().clone()
    for _ in range(3):
        assert torch.equal(first, s.run())


def test_refusals_on_the_device():
    from gogguf_b200.csrc import fast_attention as A
    from gogguf_b200.csrc.build import KernelError
    s = Setup(groups=[2], prefix=[2], own=(1, 9), nq=4, nkv=2, d=64)
    plan = A.PrefixPlan.of_pages(s.lists, s.lengths, PAGE, "cuda")
    with pytest.raises(KernelError, match="scratch"):
        s.run(scratch=torch.empty(100, device="cuda"))
    with pytest.raises(KernelError, match="plan of"):
        A.PrefixPlan.over(plan.words, 3)
    with pytest.raises(KernelError, match="shares"):
        s.run(plan=plan, shares=9)
    with pytest.raises(KernelError, match="runs"):
        s.run(plan=plan, runs=297)
    with pytest.raises(KernelError, match="plan"):
        s.run(plan=A.PrefixPlan.of_pages(s.lists, s.lengths, PAGE, "cpu"))
    with pytest.raises(KernelError, match="sink"):
        s.run(sink=torch.zeros(3, device="cuda"))
    with pytest.raises(KernelError, match="gate"):
        s.run(gate=torch.zeros(2, 8, dtype=torch.bfloat16, device="cuda"))
    s.q = s.q.float()
    with pytest.raises(KernelError, match="bfloat16"):
        s.run()


def test_debug_build_checks_page_tables():
    """GOGGUF_B200_DEBUG=1: pages beyond the pool are recorded and not read."""
    import os
    import subprocess
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    p = subprocess.run([sys.executable, os.path.join(root, "tests", "debug_shared_script.py"), root], env=dict(os.environ, GOGGUF_B200_DEBUG="1"),
                       capture_output=True, text=True, timeout=600)
    assert p.returncode == 0 and "debug shared ok" in p.stdout, p.stdout[-2000:] + p.stderr[-4000:]
