"""Cases of the operators behind several answers to one prompt: decode attention whose sequences share the pages of a
prefix, and the shaping of logits (penalties, biases, grammar masks) before a token is drawn.

Attention: token rows of one decode step, in groups that read the same leading pages of the cache and go on in pages of their
own.  Logits: rows of a model's head, with each row's last ids, its own biases and its own row of a table of allowed ids.
"""
import math

import torch

own = False

PAGE = 64


# ---------------------------------------------------------------------------------------------------------------- cases
def _attention(name, groups, prefix_pages, own_tokens, heads, kv_heads, dim, value_dim, sink=False):
    """groups: how many rows share each prefix, as a text ("8" or "5,3,1"; a row alone has pages of its own only)."""
    return {"name": name, "op": "attention", "groups": groups, "prefix_pages": prefix_pages, "own_tokens": own_tokens,
            "heads": heads, "kv_heads": kv_heads, "dim": dim, "value_dim": value_dim, "sink": sink}


def _logits(name, rows, vocab, window, biases, masks, repeat, frequency, presence):
    """window: how many of a row's last ids count; biases: ids with a bias per row; masks: rows of the table of allowed
    ids (0: no grammar)."""
    return {"name": name, "op": "logits", "rows": rows, "vocab": vocab, "window": window, "biases": biases, "masks": masks,
            "repeat": repeat, "frequency": frequency, "presence": presence}


def listed():
    return [
        # two answers to a short question, right after it: what a step takes at the least
        _attention("two_answers_short", "2", 8, 3, 16, 8, 64, 64),
        # eight answers to a prompt of 2,048 tokens, 32 query and 8 key/value heads of 128 (the benchmark's shape and batch)
        _attention("eight_answers_2k", "8", 32, 300, 32, 8, 128, 128),
        # sixty-four answers to a prompt of 2,048 tokens, some of them long by now
        _attention("batch64_2k", "64", 32, 500, 32, 8, 128, 128),
        # sixty-four questions about one long document
        _attention("batch64_32k", "64", 512, 200, 32, 8, 128, 128),
        # three prompts in one batch, each with several answers, and rows that share nothing; heads of 80 and 72, sinks
        _attention("three_prompts_ragged", "13,7,3,1,1", 37, 130, 24, 4, 80, 72, sink=True),
        # all query heads on one key/value head of each half, a document of 16,384 tokens, a dozen readers
        _attention("twelve_readers_16k", "12", 256, 64, 32, 2, 128, 128),
        # one sequence's next token: penalties over the last 64 ids and a few biases
        _logits("one_row_penalties", 1, 151936, 64, 8, 0, 1.1, 0.2, 0.1),
        # a batch of eight inside a grammar
        _logits("eight_rows_grammar", 8, 151936, 64, 16, 12, 1.1, 0.2, 0.1),
        # sixty-four answers in different states of a grammar, penalties over a few hundred ids
        _logits("batch64_grammar", 64, 151936, 512, 32, 100, 1.05, 0.3, 0.0),
        # an odd vocabulary and the whole history of long answers
        _logits("odd_vocabulary_long_window", 13, 50257, 4096, 100, 5, 1.2, 0.05, 0.5),
        # the widest step that is replayed as a graph
        _logits("batch256_grammar", 256, 151936, 64, 4, 256, 1.0, 0.4, 0.4),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    if rng.random() < 0.5:
        while True:
            kv_heads = rng.choice([1, 2, 4, 8])
            heads = kv_heads * rng.choice([1, 2, 3, 4, 5, 8, 16])
            dim = rng.choice([64, 128, 128, 32, 72, 80, 96, 112])
            value_dim = dim if rng.random() < 0.7 else rng.choice([64, 128, 40, 88, 120])
            groups = [_log_int(rng, 2, 64)]
            while rng.random() < 0.4 and len(groups) < 4:
                groups.append(_log_int(rng, 1, 24))
            case = _attention("", ",".join(map(str, groups)), _log_int(rng, 1, 512), _log_int(rng, 1, 700), heads, kv_heads, dim,
                              value_dim, sink=rng.random() < 0.3)
            del case["name"]
            most = work(_attention("", "64", 512, 200, 32, 8, 128, 128))
            now = work(case)
            if heads <= 64 and now["flops"] <= most["flops"] and now["bytes"] <= most["bytes"]:
                return case
    vocab = rng.choice([151936, 50257, 32000, 128256, _log_int(rng, 300, 160000)])
    rows = _log_int(rng, 1, 200)
    case = _logits("", rows, vocab, _log_int(rng, 1, 8192), _log_int(rng, 1, 300) if rng.random() < 0.8 else 0,
                   _log_int(rng, 1, 200) if rng.random() < 0.7 else 0, rng.choice([1.0, 1.05, 1.3, 0.9]),
                   rng.choice([0.0, 0.1, 0.7, -0.2]), rng.choice([0.0, 0.25, 1.0]))
    del case["name"]
    case["biases"] = min(case["biases"], vocab // 2)
    return case


# --------------------------------------------------------------------------------------------------------------- inputs
def _attention_layout(case, seed):
    """Which pages each row reads, and how far: page lists (shared ones first) and the rows' positions."""
    g = torch.Generator().manual_seed(seed)
    pages = case["prefix_pages"]
    lists, positions, shared, need = [], [], [], 0
    for i, n in enumerate(int(x) for x in case["groups"].split(",")):
        # later prompts of a batch are of other lengths
        here = pages if i == 0 else max(1, int(pages * torch.rand(1, generator=g).item()))
        prefix = list(range(need, need + here))
        need += here
        for _ in range(n):
            tokens = int(torch.randint(1, case["own_tokens"] + 1, (1,), generator=g).item())
            mine = -(-tokens // PAGE)
            lists.append(prefix + list(range(need, need + mine)))
            need += mine
            positions.append(here * PAGE + tokens - 1)
            shared.append(here if n > 1 else 0)
    ids = torch.randperm(need, generator=g)
    order = torch.randperm(len(lists), generator=g).tolist()       # a batch's rows stand in any order
    lists = [ids[torch.tensor(lists[r])].tolist() for r in order]
    return lists, [positions[r] for r in order], [shared[r] for r in order], need


def _attention_data(case, seed):
    lists, positions, shared, n_pages = _attention_layout(case, seed)
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    nkv, d, dv, nq = case["kv_heads"], case["dim"], case["value_dim"], case["heads"]
    k = torch.randn(n_pages, nkv, PAGE, d, generator=g, device=dev, dtype=torch.bfloat16)
    v = torch.randn(n_pages, nkv, PAGE, dv, generator=g, device=dev, dtype=torch.bfloat16)
    q = (torch.randn(len(lists), nq * d, generator=g, device=dev) * 1.5).to(torch.bfloat16)
    sink = torch.randn(nq, generator=g, device=dev) if case["sink"] else None
    return lists, positions, shared, k, v, q, sink


def _logits_data(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    R, V, n = case["rows"], case["vocab"], case["window"]
    x = torch.randn(R, V, generator=g, device=dev) * 3.0
    # a text repeats itself: ids lie dense at the front of the vocabulary
    hist = (torch.rand(R, n, generator=g, device=dev) ** 3 * V).to(torch.int32).clamp_(max=V - 1)
    length = torch.randint(max(1, n // 2), n + 1, (R,), generator=g, device=dev, dtype=torch.int32)
    nb = case["biases"]
    ids = torch.stack([torch.randperm(V, generator=g, device=dev)[:nb] for _ in range(R)]).to(torch.int32) if nb else None
    value = torch.randn(R, nb, generator=g, device=dev) * 4.0 if nb else None
    masks = rows = None
    if case["masks"]:
        words = -(-V // 32)
        # states that allow nearly all, about half, and nearly none of the ids
        bits = torch.randint(-2 ** 31, 2 ** 31, (3, case["masks"], words), generator=g, device=dev, dtype=torch.int64).to(torch.int32)
        kind = (torch.arange(case["masks"], device=dev) % 3)[:, None]
        masks = torch.where(kind == 0, bits[0] | bits[1] | bits[2], torch.where(kind == 1, bits[0], bits[0] & bits[1] & bits[2])).contiguous()
        rows = torch.randint(0, case["masks"], (R,), generator=g, device=dev, dtype=torch.int32)
        if R > 2:
            rows[1] = -1                                      # a request without a grammar in the same batch
    return x, hist, length, ids, value, masks, rows


def prepare(case, seed):
    if case["op"] == "attention":
        lists, positions, shared, k, v, q, sink = _attention_data(case, seed)
        dev = q.device
        B, width = len(lists), max(map(len, lists))
        table = torch.tensor([p + [0] * (width - len(p)) for p in lists], dtype=torch.int32, device=dev)
        state = {"case": case, "q": q, "k": k, "v": v, "sink": sink, "table": table,
                 "positions": torch.tensor(positions, dtype=torch.int32, device=dev),
                 "rows": torch.arange(B, dtype=torch.int32, device=dev),
                 "out": torch.empty(B, case["heads"] * case["value_dim"], dtype=torch.bfloat16, device=dev)}
        groups = {}
        for r, n in enumerate(shared):
            groups.setdefault((tuple(lists[r][:n]) if n else ("alone", r)), []).append(r)
        state["groups"] = [(torch.tensor(rows, device=dev), len(key) if key[0] != "alone" else 0) for key, rows in groups.items()]
        if own:
            from gogguf_b200.csrc import fast_attention as A
            state["plan"] = A.PrefixPlan.of_pages(lists, [p + 1 for p in positions], PAGE, device=dev)
            state["scratch"] = torch.empty(A.shared_scratch(B, case["heads"], case["kv_heads"], case["value_dim"]), dtype=torch.float32, device=dev)
        return state
    x, hist, length, ids, value, masks, rows = _logits_data(case, seed)
    R = case["rows"]
    state = {"case": case, "x": x, "hist": hist, "length": length, "rings": torch.arange(R, dtype=torch.int32, device=x.device),
             "masks": masks, "mask_rows": rows, "out": torch.empty_like(x), "bias": None}
    if ids is not None:
        start = torch.arange(R + 1, dtype=torch.int32, device=x.device) * ids.shape[1]
        state["bias"] = (start, ids.reshape(-1).contiguous(), value.reshape(-1).contiguous())
    return state


# ------------------------------------------------------------------------------------------------------------------ run
def _attention_plain(s):
    c = s["case"]
    nq, nkv, d, dv = c["heads"], c["kv_heads"], c["dim"], c["value_dim"]
    G, scale = nq // nkv, 1.0 / math.sqrt(d)
    out = s["out"]
    for rows, pages in s["groups"]:
        M = rows.numel()
        q = s["q"][rows].float().view(M, nkv, G, d)
        table, pos = s["table"][rows].long(), s["positions"][rows]
        last = s["table"].shape[1]
        ks, vs = s["k"][table[:, pages:last]].float(), s["v"][table[:, pages:last]].float()      # [M, own pages, nkv, 64, .]
        ks = ks.transpose(1, 2).reshape(M, nkv, -1, d)
        vs = vs.transpose(1, 2).reshape(M, nkv, -1, dv)
        so = torch.matmul(q, ks.transpose(2, 3)) * scale                                         # [M, nkv, G, own]
        at = torch.arange(ks.shape[2], device=q.device) + pages * PAGE
        so = torch.where(at[None, None, None, :] <= pos[:, None, None, None], so, torch.full_like(so, -math.inf))
        top = so.amax(-1, keepdim=True)
        if pages:
            kp = s["k"][table[0, :pages]].float().transpose(0, 1).reshape(nkv, -1, d)            # once for all members
            vp = s["v"][table[0, :pages]].float().transpose(0, 1).reshape(nkv, -1, dv)
            qp = q.transpose(0, 1).reshape(nkv, M * G, d)
            sp = torch.matmul(qp, kp.transpose(1, 2)) * scale                                    # [nkv, M G, prefix]
            topp = sp.amax(-1).view(nkv, M, G).transpose(0, 1).unsqueeze(-1)
            top = torch.maximum(top, topp)
        if s["sink"] is not None:
            sink = s["sink"].view(1, nkv, G, 1)
            top = torch.maximum(top, sink)
        eo = torch.exp(so - top)
        total = eo.sum(-1, keepdim=True)
        acc = torch.matmul(eo, vs)
        if pages:
            ep = torch.exp(sp - top.squeeze(-1).transpose(0, 1).reshape(nkv, M * G, 1))
            total = total + ep.sum(-1).view(nkv, M, G).transpose(0, 1).unsqueeze(-1)
            acc = acc + torch.matmul(ep, vp).view(nkv, M, G, dv).transpose(0, 1)
        if s["sink"] is not None:
            total = total + torch.exp(sink - top)
        out[rows] = (acc / total).to(torch.bfloat16).reshape(M, nq * dv)
    return out


def _logits_plain(s):
    c = s["case"]
    R, V, n = c["rows"], c["vocab"], c["window"]
    x = s["x"]
    seen = (torch.arange(n, device=x.device)[None, :] < s["length"][:, None]).float()
    count = torch.zeros_like(x).scatter_add_(1, s["hist"].long(), seen)
    z = torch.where(count > 0, torch.where(x > 0, x / c["repeat"], x * c["repeat"]) - (count * c["frequency"] + c["presence"]), x)
    if s["bias"] is not None:
        _, ids, value = s["bias"]
        z = z.scatter_add(1, ids.view(R, -1).long(), value.view(R, -1))
    if s["masks"] is not None:
        word = s["masks"][s["mask_rows"].clamp(min=0).long()]                                    # [R, words]
        bit = torch.arange(32, device=x.device, dtype=torch.int32)
        allowed = ((word[:, :, None] >> bit) & 1).reshape(R, -1)[:, :V] > 0
        allowed = allowed | (s["mask_rows"] < 0)[:, None]
        z = torch.where(allowed, z, torch.full_like(z, -math.inf))
    s["out"].copy_(z)
    return s["out"]


def run(s):
    c = s["case"]
    if c["op"] == "attention":
        if not own:
            return _attention_plain(s)
        from gogguf_b200.csrc import fast_attention as A
        A.attn_decode_shared(s["q"], s["k"], s["v"], s["out"], s["positions"], s["rows"], s["table"], PAGE, s["plan"], s["scratch"],
                             c["heads"], c["kv_heads"], c["dim"], 1.0 / math.sqrt(c["dim"]), sink=s["sink"], dv=c["value_dim"])
        return s["out"]
    if not own:
        return _logits_plain(s)
    from gogguf_b200.csrc import kernels as K
    K.shape_logits(s["x"], s["out"], hist=s["hist"], hist_len=s["length"], ring_rows=s["rings"], repeat=c["repeat"],
                   frequency=c["frequency"], presence=c["presence"], bias=s["bias"], masks=s["masks"], mask_rows=s["mask_rows"])
    return s["out"]


# ----------------------------------------------------------------------------------------------------------------- work
def work(case):
    if case["op"] == "attention":
        nq, nkv, d, dv = case["heads"], case["kv_heads"], case["dim"], case["value_dim"]
        lists, positions, shared, _ = _attention_layout(case, 0)
        B = len(positions)
        # every prefix is read once, whatever its readers
        prefix = {pages[0]: n * PAGE for pages, n in zip(lists, shared) if n}
        keys = sum(prefix.values()) + sum(p + 1 - n * PAGE for p, n in zip(positions, shared))
        pairs = sum(p + 1 for p in positions)
        return {"bytes": keys * nkv * (d + dv) * 2 + B * nq * (d + dv) * 2 + sum(p // PAGE + 1 for p in positions) * 4,
                "flops": 2.0 * pairs * nq * (d + dv)}
    R, V = case["rows"], case["vocab"]
    return {"bytes": R * V * 8 + R * case["window"] * 4 + R * case["biases"] * 8 + (R * -(-V // 32) * 4 if case["masks"] else 0),
            "flops": float(R * V)}


# ---------------------------------------------------------------------------------------------------------------- exact
def exact(case, seed):
    """The definitions in 64 bits, a row (and for attention a key/value head) at a time."""
    if case["op"] == "attention":
        lists, positions, _, k, v, q, sink = _attention_data(case, seed)
        nq, nkv, d, dv = case["heads"], case["kv_heads"], case["dim"], case["value_dim"]
        G = nq // nkv
        if len(lists) * nkv > 4096:
            return None
        out = torch.empty(len(lists), nq, dv, dtype=torch.float64, device=q.device)
        for r, pages in enumerate(lists):
            at = torch.tensor(pages, device=q.device)
            n = positions[r] + 1
            for h in range(nkv):
                keys = k[at, h].reshape(-1, d)[:n].double()
                values = v[at, h].reshape(-1, dv)[:n].double()
                for i in range(h * G, h * G + G):
                    score = keys @ q[r, i * d:(i + 1) * d].double() / math.sqrt(d)
                    if sink is not None:
                        weight = torch.softmax(torch.cat([score, sink[i:i + 1].double()]), 0)[:-1]
                    else:
                        weight = torch.softmax(score, 0)
                    out[r, i] = weight @ values
        return out.reshape(len(lists), nq * dv)
    x, hist, length, ids, value, masks, rows = _logits_data(case, seed)
    out = torch.empty(x.shape, dtype=torch.float64, device=x.device)
    V = case["vocab"]
    at = torch.arange(V, device=x.device)
    for r in range(case["rows"]):
        z = x[r].double()
        seen, times = torch.unique(hist[r, :int(length[r])].long(), return_counts=True)
        old = z[seen]
        new = torch.where(old > 0, old / case["repeat"], old * case["repeat"])
        z[seen] = new - case["frequency"] * times.double() - case["presence"]
        if ids is not None:
            z[ids[r].long()] += value[r].double()
        if masks is not None and int(rows[r]) >= 0:
            word = masks[int(rows[r])].long()[at // 32]
            z[(word >> (at % 32)) & 1 == 0] = -math.inf
        out[r] = z
    return out
