"""Penalties, biases and masks on rows of logits (csrc/logit_shaping.cu) against the formula in 64 bits.

Tolerance: at most five 32-bit roundings (the quotient or product, frequency c + presence, its subtraction, the bias), each half
a step, 2^-24, of a number no larger than |x| max(repeat, 1 / repeat) + |frequency| c + |presence| + |bias|."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


def make(R, V, window=0, biases=0, states=0, requests=None, seed=0, ld=None):
    g = torch.Generator().manual_seed(seed)
    Q = requests or R
    ld = ld or V
    x = (torch.randn(R, ld, generator=g) * 3)
    kw = {}
    kw["ring_rows"] = torch.randperm(Q, generator=g)[:R].to(torch.int32) if requests else None
    if window:
        h = (torch.rand(Q, window, generator=g) ** 4 * V).to(torch.int32).clamp_(max=V - 1)
        h[torch.rand(Q, window, generator=g) < 0.05] = -1            # empty places and ids of another vocabulary
        h[torch.rand(Q, window, generator=g) < 0.05] = V + 3
        kw["hist"], kw["hist_len"] = h, torch.randint(0, window + 1, (Q,), generator=g, dtype=torch.int32)
        kw["hist_len"][0] = window
    if biases:
        n = torch.randint(0, biases + 1, (Q,), generator=g)
        ids = torch.cat([torch.randperm(V, generator=g)[:int(k)] for k in n] + [torch.zeros(0, dtype=torch.int64)])
        kw["bias"] = (torch.cat([torch.zeros(1, dtype=torch.int64), n.cumsum(0)]).to(torch.int32), ids.to(torch.int32),
                      torch.randn(ids.numel(), generator=g) * 5)
    if states:
        words = -(-V // 32) + seed % 2
        kw["masks"] = torch.randint(-2 ** 31, 2 ** 31, (states, words), generator=g).to(torch.int32)
        kw["masks"][0] = 0                                            # a state that allows nothing
        kw["mask_rows"] = torch.randint(-1, states, (Q,), generator=g).to(torch.int32)
        kw["mask_rows"][0] = 0
    return x, kw


def formula(x, V, kw, repeat, frequency, presence):
    out = x.double().clone()
    room = torch.zeros_like(out)
    for r in range(x.shape[0]):
        q = int(kw["ring_rows"][r]) if kw.get("ring_rows") is not None else r
        row, size = out[r, :V], x[r, :V].double().abs() * max(repeat, 1 / repeat)
        if "hist" in kw:
            count = torch.zeros(V, dtype=torch.float64)
            for i in kw["hist"][q, :int(kw["hist_len"][q])].tolist():
                if 0 <= i < V:
                    count[i] += 1
            hit = count > 0
            old = row[hit]
            row[hit] = torch.where(old > 0, old / repeat, old * repeat) - (frequency * count[hit] + presence)
            size[hit] += abs(frequency) * count[hit] + abs(presence)
        if "bias" in kw:
            start, ids, values = kw["bias"]
            last = {}
            for e in range(int(start[q]), int(start[q + 1])):
                last[int(ids[e])] = float(values[e])
            for i, b in last.items():
                row[i] += b
                size[i] += abs(b)
        if "masks" in kw and int(kw["mask_rows"][q]) >= 0:
            bits = np.unpackbits(kw["masks"][int(kw["mask_rows"][q])].numpy().view(np.uint8), bitorder="little")[:V]
            row[torch.from_numpy(bits == 0)] = -math.inf
        room[r, :V] = 5 * 2.0 ** -24 * size
    return out, room


def to_device(kw):
    move = lambda t: t.cuda() if isinstance(t, torch.Tensor) else t
    return {k: tuple(map(move, v)) if isinstance(v, tuple) else move(v) for k, v in kw.items()}


def run(x, V, kw, in_place=False, out_ld=None, **scalars):
    from gogguf_b200.csrc import kernels as K
    dev = to_device(kw)
    logits = x.cuda()
    if in_place:
        K.shape_logits(logits[:, :V], **dev, **scalars)
        return logits.cpu()
    out = torch.full((x.shape[0], out_ld or x.shape[1]), 9.0, device="cuda")
    K.shape_logits(logits[:, :V], out[:, :V], **dev, **scalars)
    assert torch.equal(logits.cpu(), x)
    assert (out[:, V:] == 9.0).all()
    return out.cpu()


def compare(got, want, room, V):
    got, want, room = got[:, :V].double(), want[:, :V], room[:, :V]
    inf = torch.isinf(want)
    assert torch.equal(torch.isinf(got) & (got < 0), inf)
    assert ((got - want).abs()[~inf] <= room[~inf]).all()


SIZES = {
    "one id": dict(R=1, V=1, window=3, biases=1, states=2),
    "less than a word": dict(R=3, V=31, window=5, biases=4, states=3),
    "a word and one": dict(R=2, V=33, window=40, biases=33, states=3),
    "a slice": dict(R=2, V=4096, window=64, biases=20, states=4),
    "a slice and one": dict(R=5, V=4097, window=64, biases=20, states=4, seed=1),
    "odd rows": dict(R=7, V=50257, window=300, biases=100, states=5, seed=2),
    "rows apart": dict(R=4, V=1001, ld=1030, window=17, biases=9, states=3, seed=3),
    "a wide vocabulary": dict(R=3, V=151936, window=64, biases=300, states=4, seed=4),
    "a long window": dict(R=2, V=5000, window=20000, biases=0, states=0, seed=5),
    "a window beyond 65,535": dict(R=2, V=900, window=70000, biases=40, states=3, seed=7),
    "biases beyond 65,534": dict(R=3, V=30011, window=20, biases=30011, states=0, seed=9),
    "rows of many requests": dict(R=5, V=700, window=30, biases=12, states=6, requests=19, seed=6),
    "penalties alone": dict(R=3, V=9000, window=50),
    "biases alone": dict(R=3, V=9000, biases=50),
    "masks alone": dict(R=9, V=9001, states=4, seed=1),
    "nothing": dict(R=3, V=100),
}


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("size", SIZES)
def test_matches_the_formula(size, in_place):
    kw = dict(SIZES[size])
    x, parts = make(**kw)
    V = kw["V"]
    for repeat, frequency, presence in ((1.0, 0.0, 0.0), (1.3, 0.0, 0.0), (1.0, 0.3, -0.2), (0.8, -0.1, 0.6)):
        got = run(x, V, parts, in_place, repeat=repeat, frequency=frequency, presence=presence)
        compare(got, *formula(x, V, parts, repeat, frequency, presence), V)
        if in_place:
            assert torch.equal(got[:, V:], x[:, V:])


def test_rows_of_another_distance():
    x, parts = make(4, 1001, 20, 9, 3, ld=1003)
    for ld in (1001, 1004, 1030):
        compare(run(x, 1001, parts, out_ld=ld, repeat=1.2), *formula(x, 1001, parts, 1.2, 0.0, 0.0), 1001)


def test_only_the_first_rows():
    from gogguf_b200.csrc import kernels as K
    x, parts = make(6, 500, 10, 3, 2)
    out = torch.full((6, 500), 9.0, device="cuda")
    K.shape_logits(x.cuda(), out, **to_device(parts), repeat=1.5, rows=4)
    assert (out[4:] == 9.0).all()
    compare(out[:4].cpu(), *formula(x[:4], 500, parts, 1.5, 0.0, 0.0), 500)


def test_infinities_and_nan():
    """Masked places are minus infinity whatever stood there; others go through the arithmetic; an id far outside is nobody's."""
    from gogguf_b200.csrc import kernels as K
    x = torch.tensor([[math.nan, math.inf, -math.inf, 1.0, math.nan, math.inf, 2.0, -3.0]], device="cuda")
    mask = torch.tensor([[0b00001111]], dtype=torch.int32, device="cuda")
    hist = torch.tensor([[1, 2, 3, 3, -2 ** 31, 2 ** 31 - 1, 8]], dtype=torch.int32, device="cuda")
    got = K.shape_logits(x, torch.empty_like(x), hist=hist, hist_len=torch.tensor([7], dtype=torch.int32, device="cuda"), repeat=2.0,
                         frequency=0.25, presence=0.125, masks=mask, mask_rows=torch.zeros(1, dtype=torch.int32, device="cuda")).tolist()[0]
    assert math.isnan(got[0]) and got[1] == math.inf and got[2] == -math.inf and got[3] == 0.5 - 0.5 - 0.125
    assert got[4:] == [-math.inf] * 4


def test_an_id_listed_twice_and_states_outside_the_table():
    from gogguf_b200.csrc import kernels as K
    dev = dict(dtype=torch.int32, device="cuda")
    x = torch.zeros(3, 40, device="cuda")
    bias = (torch.tensor([0, 3, 3, 3], **dev), torch.tensor([5, 5, 39], **dev), torch.tensor([1.0, 2.0, 3.0], device="cuda"))
    masks = torch.full((2, 2), -1, **dev)
    got = K.shape_logits(x, bias=bias, masks=masks, mask_rows=torch.tensor([1, 2, -7], **dev)).cpu()
    assert got[0, 5] == 2.0 and got[0, 39] == 3.0 and got[0].count_nonzero() == 2
    assert (got[1] == -math.inf).all() and (got[2] == 0).all()


def test_captured_and_replayed():
    from gogguf_b200.csrc import kernels as K
    x, parts = make(5, 3000, 25, 6, 3, requests=9)
    dev, logits, out = to_device(parts), x.cuda(), torch.empty_like(x.cuda())
    K.shape_logits(logits, out, **dev, repeat=1.1, frequency=0.5)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        K.shape_logits(logits, out, **dev, repeat=1.1, frequency=0.5)
    other, more = make(5, 3000, 25, 6, 3, requests=9, seed=8)
    logits.copy_(other)
    for k in ("hist", "hist_len", "ring_rows", "mask_rows"):
        dev[k].copy_(more[k])
    parts = {**more, "bias": parts["bias"], "masks": parts["masks"]}
    graph.replay()
    compare(out.cpu(), *formula(other, 3000, parts, 1.1, 0.5, 0.0), 3000)


@pytest.mark.parametrize("rows", [1, 64])
def test_the_same_as_the_repeat_penalty(rows):
    """Where only the repeat penalty is asked for, the same bits as its own kernel."""
    from gogguf_b200.csrc import kernels as K
    x, parts = make(rows, 2000, 64, requests=rows + 3)
    dev = to_device(parts)
    a, b = x.cuda(), x.cuda()
    K.repeat_penalty(a, dev["hist"], dev["hist_len"], dev["ring_rows"], 1.3, rows)
    K.shape_logits(b, **dev, repeat=1.3)
    assert torch.equal(a, b)
