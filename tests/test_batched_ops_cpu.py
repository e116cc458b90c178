"""The batched-step operators without a GPU: what they refuse before any
launch, the tree masks, and the plain implementations the GPU tests use."""
import ctypes

import numpy as np
import pytest

import aaedn_b200 as ab
import batched_ops_ref as ref


def _refused(call, text):
    with pytest.raises(ab.AaednError) as e:
        call()
    assert e.value.rc == ab.EINVAL and text in str(e.value), str(e.value)


A = 4096  # stands for an aligned device address: refused as no device memory at the latest


def _attention(tree=False, hd=128, kv=8, heads=32, seqs=1, rows=1, pages=1, stride=1, ws=A, ws_bytes=32 << 20, scale=0.1,
               words=1, q=A, ldq=None):
    c = ab.KvCache(A, A, A, stride, pages, kv, hd)
    if tree:
        ab.attention_tree(q, c, A, A, A, words, seqs, rows, heads, scale, A, ws, ws_bytes, ldq=ldq)
    else:
        ab.attention_packed(q, c, A, A, seqs, rows, heads, scale, A, ws, ws_bytes, ldq=ldq)


@pytest.mark.parametrize("tree", [False, True])
@pytest.mark.parametrize("bad,text", [
    (dict(hd=0), "head_dim"), (dict(hd=6), "head_dim"), (dict(hd=260), "head_dim"), (dict(heads=12), "n_heads"),
    (dict(heads=8 * 65), "n_heads"), (dict(kv=0), "n_heads"), (dict(pages=0), "n_pages"), (dict(stride=0), "pt_stride"),
    (dict(ldq=100), "ldq"), (dict(ldq=32 * 128 + 2), "ldq"), (dict(scale=float("nan")), "scale"), (dict(q=None), "d_q is null"),
    (dict(q=A + 4), "aligned"), (dict(rows=1 << 25), "rows"), (dict(seqs=1 << 17), "sequences"), (dict(), "d_q"),
])
def test_attention_refusals(tree, bad, text):
    _refused(lambda: _attention(tree, **bad), text)


def test_tree_refuses_mask_words():
    _refused(lambda: _attention(True, words=0), "mask_words")
    _refused(lambda: _attention(True, words=1025), "mask_words")


@pytest.mark.parametrize("kw", [dict(seqs=0), dict(rows=0)])
def test_attention_of_nothing_is_a_no_op(kw):
    _attention(False, **kw)
    _attention(True, **kw)


def test_kv_refusals():
    one = (ctypes.c_void_p * 1)(A)
    _refused(lambda: ab.kv_copy_pages(one, 6, 4, A, A, 1), "page_floats")
    _refused(lambda: ab.kv_copy_pages(one, 8, 0, A, A, 1), "n_pages")
    _refused(lambda: ab.kv_copy_pages((ctypes.c_void_p * 1)(None), 8, 4, A, A, 1), "null")
    _refused(lambda: ab.kv_copy_pages((ctypes.c_void_p * 1)(A + 8), 8, 4, A, A, 1), "aligned")
    _refused(lambda: ab.kv_compact(one, 4, 8, 6, A, 1, A, A, A, 1, 1), "head_dim")
    _refused(lambda: ab.kv_compact(one, 4, 0, 8, A, 1, A, A, A, 1, 1), "n_kv_heads")
    _refused(lambda: ab.kv_compact(one, 4, 8, 8, A, 0, A, A, A, 1, 1), "pt_stride")
    ab.kv_copy_pages(one, 8, 4, A, A, 0)  # nothing to do
    ab.kv_compact(one, 4, 8, 8, A, 1, A, A, A, 0, 1)
    ab.kv_compact(one, 4, 8, 8, A, 1, A, A, A, 1, 0)


def test_sample_rows_refusals():
    _refused(lambda: ab.sample_rows(A, 1, 0, None, None, None, None, A, A), "vocab")
    _refused(lambda: ab.sample_rows(A, 1, 1000001, None, None, None, None, A, A), "vocab")
    _refused(lambda: ab.sample_rows(A, 1, 100, None, None, None, None, A, A, ld=99), "ld")
    _refused(lambda: ab.sample_rows(A, 1, 100, None, None, None, None, None, A), "d_u is null")
    _refused(lambda: ab.sample_rows(None, 1, 100, None, None, None, None, A, A), "d_logits is null")
    ab.sample_rows(None, 0, 100, None, None, None, None, None, None)


def test_tree_masks_match_the_plain_ones():
    rng = np.random.default_rng(1)
    for n in (1, 2, 63, 64, 65, 200):
        p = ref.random_parents(rng, n)
        assert np.array_equal(ab.tree_masks(p), ref.masks_of(p, max(1, -(-n // 64))))
    with pytest.raises(ValueError):
        ab.tree_masks([0])
    with pytest.raises(ValueError):
        ab.tree_masks([-1, 1])


def test_plain_sample_cuts():
    lg = np.log(np.array([0.1, 0.4, 0.2, 0.3], np.float32))
    assert ref.sample(lg, 0.0, 0, 1.0, 0.0, 0.9) == 1
    assert [ref.sample(lg, 1.0, 0, 1.0, 0.0, u) for u in (0.0, 0.39, 0.41, 0.69, 0.71, 0.89, 0.91)] == [1, 1, 3, 3, 2, 2, 0]
    assert ref.sample(lg, 1.0, 2, 1.0, 0.0, 0.99) == 3
    assert ref.sample(lg, 1.0, 0, 0.5, 0.0, 0.99) == 3
    assert ref.sample(lg, 1.0, 0, 1.0, 0.6, 0.99) == 3
    assert ref.sample(np.full(4, np.nan), 1.0, 0, 1.0, 0.0, 0.5) == 0
