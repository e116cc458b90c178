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


def test_a_dropped_draft_gives_its_pages_back(monkeypatch):
    """Any call that drops a draft keeps the pages of the sequence's tokens and
    of the call's own rows only."""
    bm, om = _small_rows(monkeypatch, 256, 3)
    total, free0 = bm.kv_pages()
    s = bm.open()
    p = _tokens(GQA, 260, 60)
    bm.prefill(s, p)

    def held():
        return free0 - bm.kv_pages()[1]

    def draft():
        bm.step_tree([s], [_tokens(GQA, 261, 200)], [[-1] * 200], want_logits=False)
        assert held() == 5

    draft()
    lg, _ = bm.step([s], [3])
    assert held() == 1 and _rel_err(lg[0], _run(om, p + [3])) < 1e-4
    draft()
    lg, _ = bm.prefill_batch([s], [[4, 5, 6, 7]])
    assert held() == 2 and _rel_err(lg[0], _run(om, p + [3, 4, 5, 6, 7])) < 1e-4
    draft()
    bm.step_tree([s], [[1, 2]], [[-1, 0]], want_logits=False)  # a smaller draft in its place
    assert held() == 2
    draft()
    lg, _ = bm.prefill(s, [8])
    assert held() == 2 and _rel_err(lg, _run(om, p + [3, 4, 5, 6, 7, 8])) < 1e-4
    # the pages are another sequence's at once
    draft()
    o = bm.open()
    bm.step([s], [9])
    bm.prefill(o, _tokens(GQA, 262, 64 * (total - 2)))
    assert bm.kv_pages()[1] == 0
    lg, _ = bm.step([s], [10])
    assert _rel_err(lg[0], _run(om, p + [3, 4, 5, 6, 7, 8, 9, 10])) < 1e-4
    # two sequences of one call: the first may need what the second's draft held
    bm.close_seq(o)
    bm.step_tree([s], [[1] * 200], [[-1] * 200], want_logits=False)
    o = bm.open()
    bm.prefill(o, _tokens(GQA, 263, 64 * bm.kv_pages()[1]))
    assert bm.kv_pages()[1] == 0
    bm.step([o, s], [1, 2])
    assert bm.kv_pages()[1] == 2
    bm.close()


QUIET_SYNC = """
import sys, time
sys.path[:0] = {paths!r}
import torch
import aaedn_b200 as ab
torch.zeros(1, device="cuda")
L = ab.lib()

def least(call):
    call()
    took = []
    for _ in range(30):
        t = time.perf_counter()
        for _ in range(50):
            call()
        took.append(time.perf_counter() - t)
    return min(took) / 50

a, b = least(lambda: L.aaedn_stream_sync(None)), least(lambda: L.aaedn_device_sync())
print("stream %.2f us, device %.2f us" % (a * 1e6, b * 1e6))
assert b < 2 * a + 2e-6
"""


def test_a_device_sync_reads_nothing_back_before_the_first_attention_call():
    """A wait for an idle device takes about a microsecond, a word copied from it
    about ten: in a program without packed or tree attention there is none."""
    import os
    import subprocess
    import sys
    paths = [os.path.dirname(os.path.dirname(os.path.abspath(ab.__file__)))]
    r = subprocess.run([sys.executable, "-c", QUIET_SYNC.format(paths=paths)], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stdout + r.stderr
