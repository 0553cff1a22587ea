"""Which rows of a step read a prefix together, the plan's words, and what the kernel's face refuses (no GPU)."""
import numpy as np
import pytest
import torch

from gogguf_b200.csrc import fast_attention as A
from gogguf_b200.csrc import kernels as K
from gogguf_b200.csrc.build import KernelError


def groups_of(pages, lengths, page_size=64):
    table = np.full((len(pages), max(map(len, pages))), -1)
    for r, p in enumerate(pages):
        table[r, :len(p)] = p
    got = A.shared_groups(table, [max(0, (n - 1) // page_size) for n in lengths])
    return sorted((sorted(rows), n) for rows, n in got)


def test_rows_that_share_nothing_have_no_group():
    assert groups_of([[0, 1], [2, 3]], [100, 100]) == []
    assert groups_of([[5]], [64]) == []


def test_shared_pages_end_before_every_rows_newest_position():
    # the third page is the same, too, but row 1's newest position lies in it
    assert groups_of([[7, 8, 9, 1], [7, 8, 9]], [200, 130]) == [([0, 1], 2)]
    # position 128 is the first of page 2: pages 0 and 1 lie before it
    assert groups_of([[7, 8, 9], [7, 8, 4]], [129, 129]) == [([0, 1], 2)]
    # the newest position is the last of page 1: only page 0 lies before it
    assert groups_of([[7, 8], [7, 8]], [128, 128]) == [([0, 1], 1)]
    assert groups_of([[7], [7]], [1, 64]) == []


def test_two_prompts_and_a_row_alone():
    pages = [[1, 2, 3], [4, 5, 6], [1, 2, 7], [8, 9, 10], [4, 5, 11], [1, 2, 12]]
    assert groups_of(pages, [150] * 6) == [([0, 2, 5], 2), ([1, 4], 2)]


def test_a_tree_is_cut_where_it_saves_most():
    # all six share page 1; two halves share ten pages more each: 2 * 2 * 11 reads saved against 5 * 1
    a, b = list(range(100, 110)), list(range(200, 210))
    pages = [[1] + a + [300 + i] for i in range(3)] + [[1] + b + [400 + i] for i in range(3)]
    assert groups_of(pages, [11 * 64 + 5] * 6) == [([0, 1, 2], 11), ([3, 4, 5], 11)]
    # one page more for two of six: the whole group saves 5 * 4, the pair 1 * 5
    pages = [[1, 2, 3, 4, 5, 10], [1, 2, 3, 4, 5, 11]] + [[1, 2, 3, 4, 20 + i, 30 + i] for i in range(4)]
    assert groups_of(pages, [5 * 64 + 1] * 6) == [(list(range(6)), 4)]


@pytest.mark.parametrize("seed", range(8))
def test_groups_of_random_trees_share_what_they_say(seed):
    rng = np.random.default_rng(seed)
    pages, fresh = [[0] * 0], 0
    for _ in range(40):
        p = list(pages[rng.integers(len(pages))])
        p = p[:rng.integers(len(p) + 1)]
        for _ in range(rng.integers(1, 5)):
            p.append(fresh)
            fresh += 1
        pages.append(p)
    pages = pages[1:]
    lengths = [int(rng.integers(1, 64 * len(p) + 1)) for p in pages]
    seen = set()
    for rows, n in groups_of(pages, lengths):
        assert len(rows) >= 2 and n >= 1 and not seen & set(rows)
        seen |= set(rows)
        for r in rows:
            assert pages[r][:n] == pages[rows[0]][:n] and n * 64 <= lengths[r] - 1


def test_a_long_chain_of_forks():
    """Row i shares i + 1 pages with the rows after it: a chain of two thousand forks is no deeper than Python goes."""
    n = 2000
    pages = np.full((n, n + 1), -1)
    trunk = np.arange(n)
    for r in range(n):
        pages[r, :r + 1] = trunk[:r + 1]
        pages[r, r + 1] = n + r
    got = A.shared_groups(pages, [r + 1 for r in range(n)])
    seen = [r for rows, _ in got for r in rows]
    assert len(seen) == len(set(seen)) and all((pages[rows, :k] == pages[rows[0], :k]).all() and k >= 1 for rows, k in got)


def test_plan_words():
    plan = A.PrefixPlan([([3, 0], 7), ([2], 1)], 5, "cpu")
    w = plan.words.tolist()
    assert len(w) == A.PrefixPlan.words_for(5) == 45 and w[0] == 2
    assert w[4:7] == [0, 2, 3]                      # first members
    assert w[10:12] == [7, 1]                       # pages
    assert w[15:17] == [3, 2]                       # first rows
    assert w[20:23] == [3, 0, 2]                    # rows
    assert w[25:30] == [7, 0, 1, 7, 0]              # pages of each row
    assert w[30:35] == [0, -1, 1, 0, -1]            # group of each row
    assert [w[35], w[37], w[38]] == [1, 0, 0]       # place among the members
    empty = A.PrefixPlan([], 3, "cpu").words.tolist()
    assert empty == [0] * 20 + [-1] * 3 + [0] * 3 + [0, 1, 2]


def test_rows_with_many_pages_of_their_own_come_first():
    words = np.full(A.PrefixPlan.words_for(4), 9, dtype=np.int32)
    A.PrefixPlan.pack([([0, 2], 1)], 4, words, [2, 7, 3])                 # the last row is padding
    assert words[-4:].tolist() == [1, 2, 0, 3]
    A.PrefixPlan.pack([], 4, words)
    assert words[-4:].tolist() == [0, 1, 2, 3]
    with pytest.raises(KernelError):
        A.PrefixPlan.pack([], 4, words, [1] * 5)


def test_own_pages_and_their_shares():
    assert A.PrefixPlan.of_pages([[0, 1, 2], [0, 1, 3], [5]], [140, 170, 3], 64, "cpu").own_pages == 1
    assert A.PrefixPlan.of_pages([[0, 1, 2, 7], [0, 1, 3], [5]], [193, 170, 3], 64, "cpu").own_pages == 2
    assert A.shared_shares(64, 8, 100) == 1 and A.shared_shares(2, 8, 100) == 8 and A.shared_shares(2, 8, 3) == 1 and A.shared_shares(8, 8, 9) == 4
    assert A.shared_shares(4000, 8, 100) == 1


def test_when_a_prefix_pays_and_in_how_many_runs():
    assert not A.prefix_pays([], 4, 8) and not A.prefix_pays([(2, 60)], 2, 8) and A.prefix_pays([(2, 130)], 2, 8)
    assert not A.prefix_pays([(8, 32)], 8, 8) and A.prefix_pays([(8, 64)], 8, 8) and A.prefix_pays([(64, 32)], 64, 8)
    assert A.prefix_pays([(300, 20)], 300, 8) and not A.prefix_pays([(2, 20)], 300, 8)
    assert A.shared_runs([(64, 32)], 32, 8) == 128 and A.shared_runs([(2, 3)], 32, 8) == 6 and A.shared_runs([(64, 512)], 32, 8) == 296 and A.shared_runs([], 32, 8) == 148


@pytest.mark.parametrize("groups, n", [([([0, 5], 2)], 5), ([([-1, 2], 2)], 5), ([([1, 1], 2)], 5), ([([0, 1], 2), ([1, 2], 2)], 5),
                                       ([([], 3)], 5), ([([0, 1], 0)], 5), ([], 0)])
def test_plan_refuses(groups, n):
    with pytest.raises(KernelError):
        A.PrefixPlan(groups, n, "cpu")


def test_of_pages_refuses():
    with pytest.raises(KernelError):
        A.PrefixPlan.of_pages([[0]], [65], 64, "cpu")         # 65 positions do not fit a page
    with pytest.raises(KernelError):
        A.PrefixPlan.of_pages([[0]], [1, 2], 64, "cpu")
    with pytest.raises(KernelError):
        A.PrefixPlan.of_pages([], [], 64, "cpu")
    with pytest.raises(KernelError):
        A.PrefixPlan.over(torch.zeros(39, dtype=torch.int32), 5)


def test_attention_refuses_what_is_not_on_the_device():
    t = torch.zeros(2, 8 * 64, dtype=torch.bfloat16)
    pool = torch.zeros(4, 4, 64, 64, dtype=torch.bfloat16)
    i = torch.zeros(2, dtype=torch.int32)
    plan = A.PrefixPlan([([0, 1], 1)], 2, "cpu")
    scratch = torch.zeros(A.shared_scratch(2, 8, 4, 64))
    with pytest.raises(KernelError, match="CUDA"):
        A.attn_decode_shared(t, pool, pool, t, i, i, torch.zeros(2, 2, dtype=torch.int32), 64, plan, scratch, 8, 4, 64, 0.1)
    with pytest.raises(KernelError, match="outside"):
        A.attn_decode_shared(t, pool, pool, t, i, i, torch.zeros(2, 2, dtype=torch.int32), 64, plan, scratch, 8, 4, 136, 0.1)
    with pytest.raises(KernelError):
        A.shared_scratch(2, 9, 4, 64)


LOGITS = torch.zeros(3, 40)
INT = dict(dtype=torch.int32)
BAD = {
    "dtype": dict(logits=LOGITS.double()),
    "columns apart": dict(logits=torch.zeros(3, 80)[:, ::2]),
    "out's shape": dict(out=torch.zeros(3, 41)),
    "too many rows": dict(rows=4),
    "overlap": dict(logits=torch.zeros(200)[:120].view(3, 40), out="shifted"),
    "repeat": dict(repeat=0.0),
    "repeat infinite": dict(repeat=float("inf")),
    "frequency": dict(frequency=float("nan")),
    "hist alone": dict(hist=torch.zeros(3, 4, **INT)),
    "hist's type": dict(hist=torch.zeros(3, 4, dtype=torch.int64), hist_len=torch.zeros(3, **INT)),
    "hist_len": dict(hist=torch.zeros(3, 4, **INT), hist_len=torch.zeros(2, **INT)),
    "fewer requests than rows": dict(hist=torch.zeros(2, 4, **INT), hist_len=torch.zeros(2, **INT)),
    "ring_rows": dict(hist=torch.zeros(3, 4, **INT), hist_len=torch.zeros(3, **INT), ring_rows=torch.zeros(2, **INT)),
    "masks alone": dict(masks=torch.zeros(2, 2, **INT)),
    "masks too narrow": dict(masks=torch.zeros(2, 1, **INT), mask_rows=torch.zeros(3, **INT)),
    "no masks": dict(masks=torch.zeros(0, 2, **INT), mask_rows=torch.zeros(3, **INT)),
    "bias": dict(bias=(torch.zeros(4, **INT), torch.zeros(2, **INT), torch.zeros(3))),
    "requests disagree": dict(bias=(torch.zeros(5, **INT), torch.zeros(2, **INT), torch.zeros(2)), masks=torch.zeros(2, 2, **INT),
                              mask_rows=torch.zeros(3, **INT)),
    "not on the device": dict(),
}


@pytest.mark.parametrize("case", BAD)
def test_shape_logits_refuses(case):
    kw = dict(BAD[case])
    x = kw.pop("logits", LOGITS)
    out = kw.pop("out", None)
    if isinstance(out, str):
        out = x.reshape(-1).as_strided((3, 40), (40, 1), 20)
    with pytest.raises(KernelError):
        K.shape_logits(x, out, **kw)
