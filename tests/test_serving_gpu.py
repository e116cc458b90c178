"""The batched operators together, as a server runs them on a batched model:
prompts packed into common passes, drafted trees verified in one pass, the
accepted path compacted into the cache, tokens drawn on the device. Every
result is compared with the oracle, which runs each sequence on its own.
Bars as the model tests: greedy tokens identical, logits within 1e-4."""
import numpy as np
import pytest

import aaedn_b200 as ab
import batched_ops_ref as ref
import pyoracle

pytestmark = pytest.mark.gpu

GQA = dict(dim=256, n_layers=2, n_heads=8, n_kv_heads=2, head_dim=32, ffn_dim=512, vocab=1000, max_seq=512,
           rope_theta=500000.0, eps=1e-6)
WIDE = dict(dim=512, n_layers=2, n_heads=4, n_kv_heads=2, head_dim=128, ffn_dim=512, vocab=777, max_seq=512,
            rope_theta=10000.0, eps=1e-6)


def _rel_err(a, b):
    return float(np.abs(a - b).max() / max(1e-30, np.abs(b).max()))


def _run(om, tokens):
    om.reset()
    lg = None
    for t in tokens:
        lg = om.step(int(t))
    return lg


@pytest.fixture(scope="module", params=["gqa32", "wide128"])
def pair(request):
    cfg = GQA if request.param == "gqa32" else WIDE
    w = ab.synthetic_weights(cfg, 5)
    om = pyoracle.OracleModel(pyoracle.Oracle(), cfg, w)
    bm = ab.BatchedModel(cfg, max_seqs=8, kv_tokens=8 * 256)
    bm.set_weights(w)
    yield cfg, om, bm
    bm.close()


def _tokens(cfg, stream, n):
    return [int(x) for x in ab.synth_tokens(9, stream, cfg["vocab"], n)]


def test_packed_prefill_matches_each_alone(pair):
    cfg, om, bm = pair
    lens = [5, 64, 1, 130, 33]
    seqs = [bm.open() for _ in lens]
    toks = [_tokens(cfg, 20 + i, n) for i, n in enumerate(lens)]
    logits, nxt = bm.prefill_batch(seqs, toks)
    for i in range(len(lens)):
        want = _run(om, toks[i])
        assert _rel_err(logits[i], want) < 1e-4 and int(nxt[i]) == int(np.argmax(want)), i
        assert bm.seq_len(seqs[i]) == lens[i]
    # the sequences go on, of other lengths (one of them a single token)
    more = [_tokens(cfg, 40 + i, n) for i, n in enumerate([70, 1, 64, 2, 31])]
    logits, nxt = bm.prefill_batch(seqs[::-1], more[::-1])
    for i in range(len(lens)):
        want = _run(om, toks[i] + more[i])
        assert _rel_err(logits[len(lens) - 1 - i], want) < 1e-4, i
    for s in seqs:
        bm.close_seq(s)


def test_packed_prefill_in_chunks(pair, monkeypatch):
    cfg, om, _ = pair
    monkeypatch.setenv("AAEDN_PREFILL_ROWS", "48")
    bm = ab.BatchedModel(cfg, max_seqs=6, kv_tokens=6 * 256)
    bm.set_weights(ab.synthetic_weights(cfg, 5))
    lens = [100, 7, 48, 1, 60]  # sequences cut by the chunks, and several in one
    seqs = [bm.open() for _ in lens]
    toks = [_tokens(cfg, 60 + i, n) for i, n in enumerate(lens)]
    logits, nxt = bm.prefill_batch(seqs, toks)
    for i in range(len(lens)):
        want = _run(om, toks[i])
        assert _rel_err(logits[i], want) < 1e-4 and int(nxt[i]) == int(np.argmax(want)), i
    bm.close()


def test_tree_nodes_match_their_paths_and_accept_keeps_one(pair):
    cfg, om, bm = pair
    total, free0 = bm.kv_pages()
    rng = np.random.default_rng(1)
    prompts = [_tokens(cfg, 80 + i, n) for i, n in enumerate([60, 130, 1])]
    seqs = [bm.open() for _ in prompts]
    bm.prefill_batch(seqs, prompts, want_logits=False)
    hist = [list(p) for p in prompts]
    for turn in range(3):
        counts = [int(x) for x in rng.integers(1, 14, len(seqs))]
        parents = [ref.random_parents(rng, n) for n in counts]
        drafts = [[int(t) for t in rng.integers(0, cfg["vocab"], n)] for n in counts]
        logits, nxt = bm.step_tree(seqs, drafts, parents)
        at, keep = 0, []
        for i, n in enumerate(counts):
            paths = []
            for j in range(n):
                p = parents[i][j]
                paths.append((paths[p] if p >= 0 else []) + [j])
            for j in range(n):
                want = _run(om, hist[i] + [drafts[i][x] for x in paths[j]])
                assert _rel_err(logits[at + j], want) < 1e-4, (turn, i, j)
                assert int(nxt[at + j]) == int(np.argmax(want)), (turn, i, j)
            at += n
            keep.append(max(paths, key=len) if i != turn else [])  # one sequence accepts nothing
        for i, s in enumerate(seqs):
            assert bm.seq_len(s) == len(hist[i])  # drafted nodes are no tokens yet
        bm.accept(seqs, keep)
        for i, s in enumerate(seqs):
            hist[i] += [drafts[i][x] for x in keep[i]]
            assert bm.seq_len(s) == len(hist[i])
        assert free0 - bm.kv_pages()[1] == sum(-(-len(h) // 64) for h in hist)
        # the compacted cache is that of the plain sequence
        more = [_tokens(cfg, 100 + turn, 1) for _ in seqs]
        logits, _ = bm.prefill_batch(seqs, more)
        for i in range(len(seqs)):
            hist[i] += more[i]
            assert _rel_err(logits[i], _run(om, hist[i])) < 1e-4, (turn, i)
    for s in seqs:
        bm.close_seq(s)
    assert bm.kv_pages()[1] == free0


def test_a_draft_that_is_not_accepted_leaves_nothing(pair):
    cfg, om, bm = pair
    total, free0 = bm.kv_pages()
    s = bm.open()
    p = _tokens(cfg, 120, 60)
    bm.prefill(s, p)
    bm.step_tree([s], [[1] * 30], [list(range(-1, 29))])  # over the page's end
    assert free0 - bm.kv_pages()[1] == 2
    kid = bm.fork(s)  # shares the pages of the tokens only
    assert free0 - bm.kv_pages()[1] == 1
    with pytest.raises(ab.AaednError):
        bm.accept([s], [[0]])  # the draft is gone
    lg, _ = bm.step([s, kid], [3, 4])
    assert _rel_err(lg[0], _run(om, p + [3])) < 1e-4 and _rel_err(lg[1], _run(om, p + [4])) < 1e-4
    bm.close_seq(s)
    bm.close_seq(kid)
    assert bm.kv_pages()[1] == free0


def test_trees_on_forked_sequences(pair):
    """Branches that share a partly filled page draft at the same time: each
    copies the page before its nodes are written."""
    cfg, om, bm = pair
    total, free0 = bm.kv_pages()
    root = bm.open()
    p = _tokens(cfg, 130, 100)
    bm.prefill(root, p)
    kids = [bm.fork(root) for _ in range(3)]
    drafts = [[int(t) for t in _tokens(cfg, 131 + i, 5)] for i in range(4)]
    parents = [[-1, 0, 0, 1, 3], [-1, -1, 1, 2, 3], [-1, 0, 1, 2, 3], [-1, -1, -1, 0, 1]]
    bm.step_tree([root] + kids, drafts, parents)
    keep = [[0, 1, 3, 4], [1, 2, 3, 4], [0, 1], [2]]
    bm.accept([root] + kids, keep)
    lg, _ = bm.step([root] + kids, [5, 6, 7, 8])
    for i in range(4):
        want = _run(om, p + [drafts[i][x] for x in keep[i]] + [5 + i])
        assert _rel_err(lg[i], want) < 1e-4, i
    for s in [root] + kids:
        bm.close_seq(s)
    assert bm.kv_pages()[1] == free0


def test_sampled_steps_draw_from_their_logits(pair):
    cfg, om, bm = pair
    rng = np.random.default_rng(3)
    seqs = [bm.open() for _ in range(6)]

    def draw(n):
        return dict(temperature=rng.choice([0.0, 0.7, 1.0], n), top_k=rng.choice([0, 20], n), top_p=rng.choice([1.0, 0.9], n),
                    min_p=rng.choice([0.0, 0.05], n), u=rng.random(n).astype(np.float32))

    def check(logits, nxt, s):
        for i in range(len(nxt)):
            want = ref.sample(logits[i], s["temperature"][i], s["top_k"][i], s["top_p"][i], s["min_p"][i], s["u"][i])
            assert int(nxt[i]) == want, i

    s = draw(6)
    logits, nxt = bm.prefill_batch(seqs, [_tokens(cfg, 140 + i, 3 + 20 * i) for i in range(6)], sampling=s)
    check(logits, nxt, s)
    for _ in range(3):
        s = draw(6)
        logits, nxt = bm.step_sample(seqs, nxt, s, want_logits=True)
        check(logits, nxt, s)
    # more nodes than the logits buffer has rows
    s = draw(30)
    logits, nxt = bm.step_tree(seqs[:3], [[1] * 10] * 3, [[-1] * 10] * 3, sampling=s)
    check(logits, nxt, s)
    # one value for every row, and only u
    logits, nxt = bm.step_sample(seqs[3:], [1, 2, 3], dict(u=0.5), want_logits=True)
    assert [int(x) for x in nxt] == [ref.sample(x, 1.0, 0, 1.0, 0.0, 0.5) for x in logits]
    for x in seqs:
        bm.close_seq(x)


def test_greedy_drafts_of_the_model_itself_are_all_accepted(pair):
    """A drafted chain of the model's own greedy tokens verifies completely."""
    cfg, om, bm = pair
    s = bm.open()
    p = _tokens(cfg, 150, 40)
    _, first = bm.prefill(s, p)
    chain, toks = [], [first]
    for _ in range(8):
        toks.append(int(np.argmax(_run(om, p + toks))))
    _, nxt = bm.step_tree([s], [toks], [list(range(-1, 8))], want_logits=False)
    for i in range(8):
        assert int(nxt[i]) == toks[i + 1]
        chain.append(i)
    bm.accept([s], [chain])
    assert bm.seq_len(s) == 48
    bm.close_seq(s)


def test_refusals(pair):
    cfg, om, bm = pair
    total, free0 = bm.kv_pages()
    s = bm.open()
    bm.prefill(s, [1, 2, 3])

    def refused(call, rc=ab.EINVAL):
        with pytest.raises(ab.AaednError) as e:
            call()
        assert e.value.rc == rc, str(e.value)

    refused(lambda: bm.prefill_batch([s, s], [[1], [2]]))
    refused(lambda: bm.prefill_batch([s], [[]]))
    refused(lambda: bm.prefill_batch([s], [[cfg["vocab"]]]))
    refused(lambda: bm.prefill_batch([s], [[1] * 510]), ab.ESTATE)
    refused(lambda: bm.step_tree([s], [[1, 2]], [[-1, 1]]))
    refused(lambda: bm.step_tree([s], [[1, 2]], [[-1, -2]]))
    refused(lambda: bm.step_tree([s], [[1] * 257], [[-1] * 257]))
    refused(lambda: bm.accept([s], [[0]]), ab.ESTATE)
    bm.step_tree([s], [[1, 2, 3]], [[-1, 0, 0]])
    refused(lambda: bm.accept([s], [[1]]))
    refused(lambda: bm.accept([s], [[0, 1, 2]]))
    refused(lambda: bm.accept([s], [[3]]))
    bm.accept([s], [[0, 2]])
    assert bm.seq_len(s) == 5
    # a pool that runs out leaves every sequence as it was
    others = [bm.open() for _ in range(7)]
    refused(lambda: bm.prefill_batch(others, [[1] * 300] * 7), ab.ENOMEM)
    assert free0 - bm.kv_pages()[1] == 1
    lg, _ = bm.step([s], [7])
    assert _rel_err(lg[0], _run(om, [1, 2, 3, 1, 3, 7])) < 1e-4
    for x in [s] + others:
        bm.close_seq(x)
    with pytest.raises(ValueError):
        bm.step_sample([s], [1], dict(temperature=1.0))
