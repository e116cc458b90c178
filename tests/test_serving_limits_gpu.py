"""The batched model's drafts at the ends of their ranges: many pending drafts
accepted at once, what a rejected draft leaves behind. Bars as the model tests:
logits within 1e-4 of the oracle's."""
import numpy as np
import pytest

import aaedn_b200 as ab
import pyoracle
from test_serving_gpu import GQA, _rel_err, _run, _tokens

pytestmark = pytest.mark.gpu


def _small_rows(monkeypatch, rows, max_seqs):
    """A batched model whose passes take `rows` rows, and the oracle's."""
    monkeypatch.setenv("AAEDN_PREFILL_ROWS", str(rows))
    w = ab.synthetic_weights(GQA, 5)
    bm = ab.BatchedModel(GQA, max_seqs=max_seqs, kv_tokens=max_seqs * 192)
    bm.set_weights(w)
    return bm, pyoracle.OracleModel(pyoracle.Oracle(), GQA, w)


def test_drafts_of_many_calls_are_accepted_in_one(monkeypatch):
    """Sixteen drafts of 48 nodes, one call each of 48 rows, then one accept: its
    lists are longer than a pass."""
    bm, om = _small_rows(monkeypatch, 48, 16)
    seqs = [bm.open() for _ in range(16)]
    prompts = [_tokens(GQA, 200 + i, 5 + 9 * i) for i in range(16)]
    bm.prefill_batch(seqs, prompts, want_logits=False)
    drafts, keep = [], []
    for i, s in enumerate(seqs):
        drafts.append(_tokens(GQA, 230 + i, 48))
        if i % 4 == 0:  # a chain, kept whole: nothing moves
            parents, path = list(range(-1, 47)), list(range(48))
        elif i % 4 == 1:  # a chain behind a sibling: every row moves
            parents, path = [-1, -1] + list(range(1, 47)), list(range(1, 48))
        elif i % 4 == 2:  # every other node
            parents, path = [-1, -1] + list(range(46)), list(range(0, 48, 2))
        else:
            parents, path = list(range(-1, 47)), []
        bm.step_tree([s], [drafts[i]], [parents], want_logits=False)
        keep.append(path)
    bm.accept(seqs, keep)
    for i, s in enumerate(seqs):
        assert bm.seq_len(s) == len(prompts[i]) + len(keep[i]), i
    logits, _ = bm.step(seqs, [7 + i for i in range(16)])
    for i in range(16):
        want = _run(om, prompts[i] + [drafts[i][j] for j in keep[i]] + [7 + i])
        assert _rel_err(logits[i], want) < 1e-4, i
    bm.close()
