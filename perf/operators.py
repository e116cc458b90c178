"""Cases of the batched-serving operators: attention of packed prompt rows and of
drafted token trees over the paged K/V cache, copies and compaction of cache pages,
and sampling of many rows.

`listed()` and `draw()` give cases, `prepare()` makes their inputs, `run()` makes one
pass through an operator (in plain torch operations, or, with `own` set, through the
library), `work()` says what a pass cannot do without and `exact()` what it should
return, in 64 bits."""
import math
import os
import sys

import numpy as np
import torch

own = False

PAGE = 64  # tokens of a cache page
WORKSPACE = 32 << 20  # bytes: enough for every attention call


def _lib():
    at = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "project-aaedn_b200")
    if at not in sys.path:
        sys.path.insert(0, at)
    import aaedn_b200
    return aaedn_b200


# ------------------------------------------------------------------- cases
def listed():
    return [
        # chat turns that arrive together: a few short prompts, latency counts
        {"name": "packed_short_8b", "op": "packed", "heads": 32, "kv": 8, "hd": 128, "lens": "17,1,33,64", "pos": "0,0,0,0"},
        # one long prompt of the 7B shape (every head its own K/V)
        {"name": "packed_long_7b", "op": "packed", "heads": 32, "kv": 32, "hd": 128, "lens": "2048", "pos": "0"},
        # continuous batching: prompts and continued chats of odd lengths
        {"name": "packed_ragged_8b", "op": "packed", "heads": 32, "kv": 8, "hd": 128,
         "lens": "1000,77,513,1,1500,260,129,640", "pos": "0,1023,64,1999,300,0,777,1"},
        # the longest prompt: the 70B shape's heads over a full 4096-token context
        {"name": "packed_4096_70b", "op": "packed", "heads": 64, "kv": 8, "hd": 128, "lens": "4096", "pos": "0"},
        # the small models' narrow heads
        {"name": "packed_narrow", "op": "packed", "heads": 6, "kv": 6, "hd": 48, "lens": "200,31,248,5", "pos": "0,100,0,250"},
        # one user's drafted tree over a long cache: the cache is read once
        {"name": "tree_one_8b", "op": "tree", "heads": 32, "kv": 8, "hd": 128, "nodes": "16", "ctx": "4001"},
        # a server's step: trees of different sizes over caches of different lengths
        {"name": "tree_batch_70b", "op": "tree", "heads": 64, "kv": 8, "hd": 128,
         "nodes": "24,13,31,1,24,48,7,24,63,24,16,24,5,24,2,24",
         "ctx": "4000,2731,512,3999,1024,65,2048,3500,1000,4032,127,0,2900,3333,1,640"},
        # four branches' copy on write of their tail pages, every layer
        {"name": "fork_copy_8b", "op": "copy", "kv": 8, "hd": 128, "layers": 32, "pages": 96, "pairs": 4},
        # the accepted drafts of a batch moved to the front of their slots
        {"name": "compact_8b", "op": "compact", "kv": 8, "hd": 128, "layers": 32, "seqs": 16, "nodes": 24, "len": 150},
        # one sequence's next token at the 7B vocabulary
        {"name": "sample_one_32000", "op": "sample", "rows": 1, "vocab": 32000},
        # a batched step of the 8B shape
        {"name": "sample_32_128256", "op": "sample", "rows": 32, "vocab": 128256},
        # every node of a batch of drafted trees
        {"name": "sample_256_128256", "op": "sample", "rows": 256, "vocab": 128256},
    ]


HEADS = ((32, 32, 128), (32, 8, 128), (64, 8, 128), (8, 2, 32), (6, 6, 48), (16, 4, 64), (8, 1, 96))


def _log(rng, lo, hi):
    """A whole number in lo..hi, spread over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("packed", "packed", "tree", "tree", "copy", "compact", "sample", "sample"))
    if op == "sample":
        return {"op": op, "rows": _log(rng, 1, 200), "vocab": _log(rng, 300, 150000)}
    if op == "copy":
        return {"op": op, "kv": rng.choice((2, 6, 8, 32)), "hd": rng.choice((32, 48, 64, 128)), "layers": _log(rng, 2, 32),
                "pages": 64, "pairs": _log(rng, 1, 24)}
    if op == "compact":
        return {"op": op, "kv": rng.choice((2, 6, 8)), "hd": rng.choice((32, 48, 64, 128)), "layers": _log(rng, 2, 32),
                "seqs": _log(rng, 1, 24), "nodes": _log(rng, 2, 63), "len": _log(rng, 1, 190)}
    heads, kv, hd = rng.choice(HEADS)
    n = _log(rng, 1, 12)
    if op == "packed":
        lens = [_log(rng, 1, 2000 if n <= 4 else 600) for _ in range(n)]
        pos = [0 if rng.random() < 0.5 else _log(rng, 1, 2000) for _ in range(n)]
        return {"op": op, "heads": heads, "kv": kv, "hd": hd, "lens": ",".join(map(str, lens)), "pos": ",".join(map(str, pos))}
    nodes = [_log(rng, 1, 63) for _ in range(n)]
    ctx = [0 if rng.random() < 0.05 else _log(rng, 1, 8000 if n <= 4 else 4000) for _ in range(n)]
    return {"op": op, "heads": heads, "kv": kv, "hd": hd, "nodes": ",".join(map(str, nodes)), "ctx": ",".join(map(str, ctx))}


def _ints(text):
    return [int(x) for x in text.split(",")]


# ------------------------------------------------------------------ inputs
def _attention_state(case, g, rng):
    """Packed queries, a page pool in a shuffled order, and the call's index arrays."""
    tree = case["op"] == "tree"
    rows = _ints(case["nodes"] if tree else case["lens"])
    past = _ints(case["ctx"] if tree else case["pos"])
    H, KV, hd, S = case["heads"], case["kv"], case["hd"], len(rows)
    need = [-(-(p + r) // PAGE) for p, r in zip(past, rows)]
    stride, pages = max(need), sum(need) + 3
    order = rng.permutation(pages)
    table, at = np.zeros((S, stride), np.int32), 0
    for s in range(S):
        table[s, :need[s]] = order[at:at + need[s]]
        at += need[s]
    T = sum(rows)
    st = {"case": case, "S": S, "T": T, "H": H, "KV": KV, "hd": hd, "pages": pages, "stride": stride,
          "scale": 1.0 / math.sqrt(hd), "max_rows": max(rows), "max_keys": max(p + r for p, r in zip(past, rows))}
    # queries and keys as a trained model's: a common direction in the keys, a few wide dims
    wide = torch.ones(hd, device="cuda")
    wide[:: max(1, hd // 4)] = 4.0
    st["q"] = torch.randn(T, H * hd, device="cuda", generator=g) * 1.3
    st["k"] = torch.randn(pages, KV, PAGE, hd, device="cuda", generator=g) * wide + 0.5
    st["v"] = torch.randn(pages, KV, PAGE, hd, device="cuda", generator=g)
    st["table"] = torch.from_numpy(table).cuda()
    st["start"] = torch.from_numpy(np.concatenate([[0], np.cumsum(rows)]).astype(np.int32)).cuda()
    st["past"] = torch.tensor(past, dtype=torch.int32, device="cuda")
    st["out"] = torch.empty(T, H * hd, device="cuda")
    st["workspace"] = torch.empty(WORKSPACE, dtype=torch.uint8, device="cuda")
    if tree:  # every node hangs under an earlier one or under the prefix; its mask: itself and its ancestors
        masks = []
        for n in rows:
            m = []
            for i in range(n):
                parent = int(rng.integers(-1, i)) if i else -1
                m.append((m[parent] if parent >= 0 else 0) | (1 << i))
            masks += m
        st["mask"] = torch.from_numpy(np.array(masks, np.uint64).view(np.int64).reshape(-1, 1)).cuda()
    return st


def _pool_state(case, g, rng):
    L, KV, hd = case["layers"], case["kv"], case["hd"]
    st = {"case": case, "KV": KV, "hd": hd}
    if case["op"] == "copy":
        pages, n = case["pages"], case["pairs"]
        pick = rng.permutation(pages)[: 2 * n].astype(np.int32)
        st["src"], st["dst"], st["n"] = torch.from_numpy(pick[:n].copy()).cuda(), torch.from_numpy(pick[n:].copy()).cuda(), n
    else:
        S, nodes, length = case["seqs"], case["nodes"], case["len"]
        base = [length + 7 * i % 40 for i in range(S)]
        need = [-(-(b + nodes) // PAGE) for b in base]
        stride, pages = max(need), sum(need) + 2
        order, at = rng.permutation(pages), 0
        table = np.zeros((S, stride), np.int32)
        keep, start = [], [0]
        for s in range(S):
            table[s, :need[s]] = order[at:at + need[s]]
            at += need[s]
            n = int(rng.integers(0, min(nodes, 8) + 1))  # accepted drafts of this sequence
            keep += sorted(int(x) for x in rng.permutation(nodes)[:n])
            start.append(len(keep))
        st["S"], st["stride"] = S, stride
        st["table"] = torch.from_numpy(table).cuda()
        st["base"] = torch.tensor(base, dtype=torch.int32, device="cuda")
        st["keep"] = torch.tensor(keep + [0], dtype=torch.int32, device="cuda")
        st["start"] = torch.tensor(start, dtype=torch.int32, device="cuda")
        st["kept"] = len(keep)
    st["pages"] = pages
    # K and V of every layer: one pool each
    st["pool"] = torch.randn(2 * L, pages, KV, PAGE, hd, device="cuda", generator=g)
    st["arrays"] = [st["pool"][i] for i in range(2 * L)]
    return st


def _sample_state(case, g, rng):
    B, V = case["rows"], case["vocab"]
    st = {"case": case, "B": B, "V": V}
    # a model's logits: a wide bulk and a peaked head, of another sharpness in every row
    logits = torch.randn(B, V, device="cuda", generator=g) * 2.0
    peaks = torch.randint(0, V, (B, 20), device="cuda", generator=g)
    sharp = torch.rand(B, 1, device="cuda", generator=g) * 10.0
    logits.scatter_add_(1, peaks, sharp + torch.rand(B, 20, device="cuda", generator=g) * 4.0)
    st["logits"] = logits
    pick = lambda values: torch.tensor(values, device="cuda")[torch.from_numpy(rng.integers(0, len(values), B)).cuda()]  # noqa: E731
    st["temperature"] = pick([0.0, 0.6, 0.8, 1.0, 1.0, 1.3])
    st["top_k"] = pick([0, 0, 1, 40, 50, 1000]).to(torch.int32)
    st["top_p"] = pick([1.0, 0.95, 0.9, 0.5])
    st["min_p"] = pick([0.0, 0.0, 0.02, 0.1])
    st["u"] = torch.rand(B, device="cuda", generator=g).clamp_(max=1.0 - 2.0 ** -24)
    st["tokens"] = torch.zeros(B, dtype=torch.int32, device="cuda")
    return st


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    rng = np.random.default_rng(int(seed))
    if case["op"] in ("packed", "tree"):
        return _attention_state(case, g, rng)
    if case["op"] in ("copy", "compact"):
        return _pool_state(case, g, rng)
    return _sample_state(case, g, rng)


# -------------------------------------------------------------- plain forms
def _plain_attention(st):
    """All sequences padded to the longest: scores, mask, softmax, product, in fp32."""
    S, T, H, KV, hd, G = st["S"], st["T"], st["H"], st["KV"], st["hd"], st["H"] // st["KV"]
    start, past = st["start"].long(), st["past"].long()
    R, L = st["max_rows"], st["max_keys"]
    seq = torch.searchsorted(start[1:].contiguous(), torch.arange(T, device="cuda"), right=True)
    at = torch.arange(T, device="cuda") - start[seq]  # a row's place among its sequence's rows
    q = torch.zeros(S, R, H, hd, device="cuda")
    q[seq, at] = st["q"].view(T, H, hd)
    q = q.view(S, R, KV, G, hd).permute(0, 2, 3, 1, 4).reshape(S, KV, G * R, hd)
    key = torch.arange(L, device="cuda")
    page = st["table"].long()[:, key // PAGE]  # [S, L]; slots behind a sequence's last key are masked
    k = st["k"][page, :, key % PAGE].permute(0, 2, 1, 3)
    v = st["v"][page, :, key % PAGE].permute(0, 2, 1, 3)
    score = (torch.matmul(q, k.transpose(2, 3)) * st["scale"]).view(S, KV, G, R, L)
    row = torch.arange(R, device="cuda")
    if "mask" in st:
        bits = torch.zeros(S, R, dtype=torch.int64, device="cuda")
        bits[seq, at] = st["mask"][:, 0]
        node = key[None, :] - past[:, None]  # [S, L]
        seen = (bits[:, :, None] >> node.clamp(0, 63)[:, None, :]) & 1
        ok = (node < 0)[:, None, :] | ((seen == 1) & (node >= 0)[:, None, :] & (node < 64)[:, None, :])
    else:
        ok = key[None, None, :] <= past[:, None, None] + row[None, :, None]
    score = torch.where(ok[:, None, None], score, float("-inf"))
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(top == float("-inf"), 0.0, top))
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(S, KV, G * R, L), v).view(S, KV, G, R, hd) / torch.where(total == 0, 1.0, total)
    return o.permute(0, 3, 1, 2, 4).reshape(S, R, H * hd)[seq, at]


def _plain_copy(st):
    st["pool"][:, st["dst"].long()] = st["pool"][:, st["src"].long()]
    return st["pool"]


def _plain_compact(st):
    start, n = st["start"].long(), st["kept"]
    entry = torch.arange(n, device="cuda")
    seq = torch.searchsorted(start[1:].contiguous(), entry, right=True)
    to = st["base"].long()[seq] + entry - start[seq]
    frm = st["base"].long()[seq] + st["keep"].long()[:n]
    table = st["table"].long()
    rows = st["pool"][:, table[seq, frm // PAGE], :, frm % PAGE].clone()
    st["pool"][:, table[seq, to // PAGE], :, to % PAGE] = rows
    return st["pool"]


def _plain_sample(st):
    logits, B, V = st["logits"], st["B"], st["V"]
    order = torch.sort(logits, dim=1, descending=True, stable=True)
    greedy = st["temperature"] <= 0
    t = torch.where(greedy, 1.0, st["temperature"]).double()
    x = (order.values.double() - order.values[:, :1].double()) / t[:, None]
    p = torch.exp(x)
    rank = torch.arange(V, device="cuda")[None]
    k = st["top_k"].long()
    limit = torch.where((k <= 0) | (k > V), V, k)[:, None]
    keep = (rank < limit) & (p >= st["min_p"].double()[:, None])
    c = torch.cumsum(torch.where(keep, p, 0.0), 1)
    last = keep.sum(1, keepdim=True) - 1
    whole = c.gather(1, last)
    cut = torch.minimum((c < st["top_p"].double()[:, None] * whole).sum(1, keepdim=True), last)
    mass = c.gather(1, cut)
    pick = torch.minimum((c < st["u"].double()[:, None] * mass).sum(1, keepdim=True), cut)
    pick = torch.where(greedy[:, None], 0, pick)
    return order.indices.gather(1, pick)[:, 0].to(torch.int32)


# --------------------------------------------------------------------- run
def _own_attention(st):
    ab = _lib()
    cache = ab.KvCache(st["k"], st["v"], st["table"], st["stride"], st["pages"], st["KV"], st["hd"])
    stream = torch.cuda.current_stream().cuda_stream
    if "mask" in st:
        ab.attention_tree(st["q"], cache, st["start"], st["past"], st["mask"], 1, st["S"], st["T"], st["H"], st["scale"],
                          st["out"], st["workspace"], WORKSPACE, stream=stream)
    else:
        ab.attention_packed(st["q"], cache, st["start"], st["past"], st["S"], st["T"], st["H"], st["scale"], st["out"],
                            st["workspace"], WORKSPACE, stream=stream)
    return st["out"]


def _own_pool(st):
    ab = _lib()
    stream = torch.cuda.current_stream().cuda_stream
    if st["case"]["op"] == "copy":
        ab.kv_copy_pages(st["arrays"], st["KV"] * PAGE * st["hd"], st["pages"], st["src"], st["dst"], st["n"], stream=stream)
    else:
        ab.kv_compact(st["arrays"], st["pages"], st["KV"], st["hd"], st["table"], st["stride"], st["base"], st["keep"],
                      st["start"], st["S"], st["kept"], stream=stream)
    return st["pool"]


def _own_sample(st):
    ab = _lib()
    ab.sample_rows(st["logits"], st["B"], st["V"], st["temperature"], st["top_k"], st["top_p"], st["min_p"], st["u"],
                   st["tokens"], stream=torch.cuda.current_stream().cuda_stream)
    return st["tokens"]


def run(state):
    op = state["case"]["op"]
    if own:
        return (_own_attention if op in ("packed", "tree") else _own_sample if op == "sample" else _own_pool)(state)
    return (_plain_attention if op in ("packed", "tree") else _plain_sample if op == "sample"
            else _plain_copy if op == "copy" else _plain_compact)(state)


# -------------------------------------------------------------------- work
def work(case):
    op = case["op"]
    if op == "sample":
        return {"bytes": case["rows"] * (case["vocab"] * 4.0 + 24), "flops": 0.0}
    if op == "copy":
        return {"bytes": 2.0 * 2 * case["layers"] * case["pairs"] * case["kv"] * PAGE * case["hd"] * 4, "flops": 0.0}
    if op == "compact":  # on average half of min(nodes, 8) drafts of a sequence are kept
        return {"bytes": 2.0 * 2 * case["layers"] * case["seqs"] * min(case["nodes"], 8) / 2 * case["kv"] * case["hd"] * 4,
                "flops": 0.0}
    H, KV, hd = case["heads"], case["kv"], case["hd"]
    if op == "packed":
        rows, past = _ints(case["lens"]), _ints(case["pos"])
        pairs = sum(n * p + n * (n + 1) / 2 for n, p in zip(rows, past))
    else:  # a node sees the prefix, itself and a few ancestors
        rows, past = _ints(case["nodes"]), _ints(case["ctx"])
        pairs = sum(n * (p + 1) for n, p in zip(rows, past))
    keys = sum(n + p for n, p in zip(rows, past))
    return {"bytes": 4.0 * hd * (2 * H * sum(rows) + 2 * KV * keys), "flops": 4.0 * hd * H * pairs}


# ------------------------------------------------------------------- exact
def _exact_attention(st):
    H, KV, hd, G = st["H"], st["KV"], st["hd"], st["H"] // st["KV"]
    start, past, table = st["start"].tolist(), st["past"].tolist(), st["table"].cpu().numpy()
    out = torch.zeros(st["T"], H, hd, dtype=torch.float64, device="cuda")
    for s in range(st["S"]):
        n, c = start[s + 1] - start[s], past[s]
        pages = torch.from_numpy(table[s, : -(-(c + n) // PAGE)].astype(np.int64)).cuda()
        # what row i of the sequence may see
        see = torch.zeros(n, c + n, dtype=torch.bool, device="cuda")
        see[:, :c] = True
        if "mask" in st:
            words = st["mask"][start[s]:start[s + 1], 0].cpu().numpy().view(np.uint64)
            tri = np.array([[(int(w) >> j) & 1 for j in range(n)] for w in words], bool).reshape(n, n)
            see[:, c:] = torch.from_numpy(tri).cuda()
        else:
            see[:, c:] = torch.ones(n, n, dtype=torch.bool, device="cuda").tril()
        for h in range(KV):
            kd = st["k"][pages, h].reshape(-1, hd)[: c + n].double()
            vd = st["v"][pages, h].reshape(-1, hd)[: c + n].double()
            for j in range(h * G, (h + 1) * G):
                qd = st["q"][start[s]:start[s + 1], j * hd:(j + 1) * hd].double()
                e = (qd @ kd.T) * st["scale"]
                e.masked_fill_(~see, -math.inf)
                out[start[s]:start[s + 1], j] = torch.softmax(e, 1) @ vd
    return out.view(st["T"], H * hd)


def _exact_pool(st):
    pool = st["pool"].double()
    if st["case"]["op"] == "copy":
        for a, b in zip(st["src"].tolist(), st["dst"].tolist()):
            pool[:, b] = pool[:, a].clone()
        return pool
    base, keep, start, table = (st[x].tolist() for x in ("base", "keep", "start", "table"))
    for s in range(st["S"]):
        for i, node in enumerate(keep[start[s]:start[s + 1]]):
            a, b = base[s] + node, base[s] + i
            pool[:, table[s][b // PAGE], :, b % PAGE] = pool[:, table[s][a // PAGE], :, a % PAGE].clone()
    return pool


def _exact_sample(st):
    rows = [st[x].cpu().numpy() for x in ("logits", "temperature", "top_k", "top_p", "min_p", "u")]
    got = []
    for lg, t, k, tp, mp, u in zip(*rows):
        ids = np.lexsort((np.arange(lg.size), -lg.astype(np.float64)))
        if t <= 0:
            got.append(ids[0])
            continue
        n = lg.size if k <= 0 else min(int(k), lg.size)
        w = np.exp((lg[ids[:n]].astype(np.float64) - float(lg[ids[0]])) / float(t))
        w = w[w >= float(mp)]
        c = np.cumsum(w)
        c = c[: int(np.searchsorted(c, float(tp) * c[-1], side="left")) + 1]
        got.append(ids[min(int(np.searchsorted(c, float(u) * c[-1], side="left")), c.size - 1)])
    return torch.from_numpy(np.array(got, np.int32))


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] in ("packed", "tree"):
        return _exact_attention(st)
    return _exact_sample(st) if case["op"] == "sample" else _exact_pool(st)
