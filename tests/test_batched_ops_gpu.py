"""The batched-step operators on the GPU against plain 64-bit implementations:
attention of packed rows and of drafted trees over the paged cache, page
copies, compaction, sampling of many rows."""
import ctypes

import numpy as np
import pytest

import aaedn_b200 as ab
import batched_ops_ref as ref
from gpu_util import dev, empty_f32, host

pytestmark = pytest.mark.gpu


def _workspace():
    import torch
    return torch.full((ab.ATTN_ROWS_WORKSPACE_BYTES,), 0xFF, dtype=torch.uint8, device="cuda")


def _call(c, kind, masks=None, words=1, stream=None, tail=3, ldq_pad=0):
    """One call; (out [T][H hd], the rows behind the last sequence)."""
    import torch
    n = c.H * c.hd
    q = np.full((c.T + tail, n + ldq_pad), np.nan, np.float32)
    q[: c.T, :n] = c.q
    out = torch.full((c.T + tail, n + ldq_pad), 7.0, device="cuda")
    cache = ab.KvCache(dev(c.k), dev(c.v), dev(c.table), c.stride, c.n_pages, c.KV, c.hd)
    args = (dev(c.start), dev(np.array(c.past, np.int32)))
    ws, dq = _workspace(), dev(q)
    if kind == "packed":
        ab.attention_packed(dq, cache, *args, len(c.past), c.T + tail, c.H, c.scale, out, ws, ldq=n + ldq_pad,
                            ldo=n + ldq_pad, stream=stream)
    else:
        dm = dev(np.concatenate([masks, np.zeros((tail, words), np.uint64)]).view(np.int64))
        ab.attention_tree(dq, cache, *args, dm, words, len(c.past), c.T + tail, c.H, c.scale, out, ws, ldq=n + ldq_pad,
                          ldo=n + ldq_pad, stream=stream)
    ab.device_sync()
    o = host(out)
    assert np.all(o[c.T:] == 7.0) and np.all(o[:, n:] == 7.0)  # rows of no sequence, columns behind the heads
    return o[: c.T, :n]


def _check(c, kind, got, masks=None):
    want, tol = ref.attention(kind, c.q, c.k, c.v, c.table, c.start, c.past, c.H, c.scale, masks)
    bad = ~(np.abs(got - want) <= tol)
    assert not bad.any(), (bad.mean(), np.argwhere(bad)[:3], np.nanmax(np.abs(got - want)[bad]))


HEADS = [(8, 2, 128), (4, 4, 128), (8, 8, 64), (8, 2, 32), (6, 6, 48), (8, 1, 96), (6, 2, 128), (3, 1, 4), (4, 2, 256),
         (5, 1, 80)]


@pytest.mark.parametrize("H,KV,hd", HEADS)
@pytest.mark.parametrize("rows,past", [
    ([1], [0]), ([64, 1, 65], [0, 63, 64]), ([130, 7, 33, 2], [0, 100, 1, 190]), ([200], [57]),
])
def test_packed(H, KV, hd, rows, past):
    c = ref.Case(H, KV, hd, rows, past, seed=hd + H + len(rows))
    _check(c, "packed", _call(c, "packed"))


@pytest.mark.parametrize("H,KV,hd", HEADS)
@pytest.mark.parametrize("rows,past", [([1, 5, 24], [0, 63, 300]), ([63, 1, 16, 2], [130, 1, 0, 64]), ([100, 70], [37, 0])])
def test_tree(H, KV, hd, rows, past):
    c = ref.Case(H, KV, hd, rows, past, seed=3 * hd + H + len(rows))
    rng = np.random.default_rng(5)
    words = 2
    masks = np.concatenate([ref.masks_of(ref.random_parents(rng, n), words) for n in rows])
    _check(c, "tree", _call(c, "tree", masks, words), masks)


def test_long_rows_and_a_long_cache():
    c = ref.Case(2, 1, 128, [300, 3], [700, 3000], seed=11)
    _check(c, "packed", _call(c, "packed"))
    c = ref.Case(8, 1, 64, [20], [6000], seed=12)
    masks = ref.masks_of(ref.random_parents(np.random.default_rng(2), 20), 1)
    _check(c, "tree", _call(c, "tree", masks), masks)


def test_many_short_sequences():
    rng = np.random.default_rng(4)
    rows = [int(x) for x in rng.integers(1, 4, 150)]
    past = [int(x) for x in rng.integers(0, 70, 150)]
    c = ref.Case(4, 2, 64, rows, past, seed=13)
    _check(c, "packed", _call(c, "packed"))


def test_sequences_without_rows():
    c = ref.Case(4, 2, 64, [0, 5, 0, 0, 70, 0], [10, 3, 0, 64, 1, 5], seed=14)
    _check(c, "packed", _call(c, "packed"))


def test_rows_that_attend_nothing_are_zero():
    c = ref.Case(4, 2, 128, [9, 4], [0, 0], seed=15)
    masks = np.zeros((13, 1), np.uint64)
    masks[3] = 0b1010
    masks[10] = 0b10
    got = _call(c, "tree", masks)
    _check(c, "tree", got, masks)
    assert np.all(got[[0, 1, 2, 12]] == 0)


def test_mask_bits_of_absent_nodes_are_ignored():
    c = ref.Case(4, 2, 64, [3, 2], [70, 5], seed=16)
    masks = np.full((5, 1), (1 << 64) - 1, np.uint64)
    _check(c, "tree", _call(c, "tree", masks), masks)


@pytest.mark.parametrize("hd", [64, 128])
def test_values_of_any_size(hd):
    """K, V and q far from 1 in both directions, and K/V rows of very different
    sizes within a page."""
    for fk, fq, fv in ((1e-6, 1e5, 1e-8), (3e4, 1e-5, 1e7), (1e10, 1e-10, 1e20)):
        c = ref.Case(4, 2, hd, [40, 3], [100, 9], seed=17)
        c.k *= np.float32(fk)
        c.q *= np.float32(fq)
        c.v *= np.float32(fv)
        _check(c, "packed", _call(c, "packed"))
    c = ref.Case(4, 2, hd, [40, 3], [100, 9], seed=18)
    with np.errstate(invalid="ignore"):
        c.v *= np.float32(10.0) ** np.random.default_rng(1).integers(-4, 1, (c.n_pages, 1, 64, 1)).astype(np.float32)
    _check(c, "packed", _call(c, "packed"))


@pytest.mark.parametrize("hd", [48, 128, 256])
def test_infinities_and_nan_reach_the_rows_that_attend_them_only(hd):
    c = ref.Case(4, 2, hd, [30, 20], [70, 64], seed=19)
    page, row = c.table[0, 80 // 64], 80 % 64  # slot 80 of sequence 0 is its row 10
    for arr, value in ((c.k, np.nan), (c.v, np.nan), (c.v, np.inf)):
        keep = arr[page, 1, row, 3]
        arr[page, 1, row, 3] = value
        got = _call(c, "packed")
        arr[page, 1, row, 3] = keep
        want, tol = ref.attention("packed", c.q, c.k, c.v, c.table, c.start, c.past, c.H, c.scale)
        hit = np.zeros_like(got, bool)
        hit[10:30, 2 * hd: 4 * hd] = True  # the heads of K/V head 1, rows at and behind the slot
        assert np.all(np.abs(got - want)[~hit] <= tol[~hit])
        touched = (~np.isfinite(got[10:30])).reshape(20, 4, hd).any(2)
        assert np.all(touched[:, 2:]), touched
    c.q[7] = np.nan
    got = _call(c, "packed")
    want, tol = ref.attention("packed", np.nan_to_num(c.q), c.k, c.v, c.table, c.start, c.past, c.H, c.scale)
    rest = np.arange(c.T) != 7
    assert np.all(np.abs(got - want)[rest] <= tol[rest]) and np.all(np.isnan(got[7]))


@pytest.mark.parametrize("hd", [64, 128, 256])
def test_pages_outside_the_pool_and_slots_behind_the_table_are_left_out(hd):
    c = ref.Case(4, 2, hd, [10, 5], [200, 130], seed=20, poison=False)
    c.table[0, 1] = -3
    c.table[1, 0] = c.n_pages + 5
    _check(c, "packed", _call(c, "packed"))
    c.past[1] = 64 * c.stride + 10  # every row of it behind the table
    got = _call(c, "packed")
    # the slots the table has
    n = c.start[2] - c.start[1]
    full = ref.attention("packed", c.q, c.k, c.v, c.table, c.start, c.past, c.H, c.scale)
    assert n == 5 and np.all(np.abs(got - full[0]) <= full[1])


def test_strides_stream_and_repeats():
    import torch
    c = ref.Case(8, 2, 128, [100, 9, 40], [3, 500, 0], seed=21)
    want, tol = ref.attention("packed", c.q, c.k, c.v, c.table, c.start, c.past, c.H, c.scale)
    first = _call(c, "packed", ldq_pad=12)
    assert np.all(np.abs(first - want) <= tol)
    st = torch.cuda.Stream()
    torch.cuda.synchronize()
    again = _call(c, "packed", ldq_pad=12, stream=st.cuda_stream)
    assert np.array_equal(first, again)  # no atomics: the same bits every time


def test_captured_and_replayed_with_other_lengths():
    import torch
    c = ref.Case(8, 2, 128, [60, 4], [200, 80], seed=22, poison=False)
    n = c.H * c.hd
    q, k, v, table = dev(c.q), dev(c.k), dev(c.v), dev(c.table)
    start, past = dev(c.start), dev(np.array(c.past, np.int32))
    out = empty_f32(c.T * n)
    ws = _workspace()
    cache = ab.KvCache(k, v, table, c.stride, c.n_pages, c.KV, c.hd)
    st = torch.cuda.Stream()
    g = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.stream(st):
        g.capture_begin()
        ab.attention_packed(q, cache, start, past, 2, c.T, c.H, c.scale, out, ws, stream=st.cuda_stream)
        g.capture_end()
    for new_past, new_start in (([200, 80], [0, 60, 64]), ([5, 100], [0, 10, 64]), ([0, 0], [0, 64, 64])):
        past.copy_(torch.tensor(new_past, dtype=torch.int32))
        start.copy_(torch.tensor(new_start, dtype=torch.int32))
        g.replay()
        ab.device_sync()
        got = host(out).reshape(c.T, n)
        want, tol = ref.attention("packed", c.q, c.k, c.v, c.table, new_start, new_past, c.H, c.scale)
        assert np.all(np.abs(got - want) <= tol)


def test_index_arrays_that_make_no_sense_stay_in_bounds():
    """Descending starts, negative lengths, rows past the end: no requirement
    on the values, only that the call returns and rows in no sequence stay."""
    import torch
    c = ref.Case(4, 2, 128, [20, 20], [64, 10], seed=23, poison=False)
    for start, past in (([0, 30, 20], [64, 10]), ([5, 10, 4000], [-7, -100]), ([-3, 8, 40], [2**31 - 1, 5]),
                        ([40, 20, 0], [0, 0]), ([2**31 - 1, -2**31, 7], [1, 1])):
        out = torch.full((40, c.H * c.hd), 7.0, device="cuda")
        cache = ab.KvCache(dev(c.k), dev(c.v), dev(c.table), c.stride, c.n_pages, c.KV, c.hd)
        ab.attention_packed(dev(c.q), cache, dev(np.array(start, np.int32)), dev(np.array(past, np.int32)), 2, 40, c.H,
                            c.scale, out, _workspace())
        ab.device_sync()


@pytest.mark.parametrize("H,KV,hd", [(64, 1, 16), (33, 1, 128), (64, 1, 192), (45, 15, 68)])
def test_any_number_of_heads_on_a_kv_head(H, KV, hd):
    c = ref.Case(H, KV, hd, [5, 1, 17], [70, 0, 3], seed=24)
    _check(c, "packed", _call(c, "packed"))


@pytest.mark.parametrize("hd", [32, 128, 160])
@pytest.mark.parametrize("scale", [0.0, -0.2, 3.0])
def test_scales(hd, scale):
    c = ref.Case(4, 2, hd, [70, 3], [5, 80], seed=25)
    c.scale = scale
    _check(c, "packed", _call(c, "packed"))


@pytest.mark.parametrize("hd", [64, 128, 160])
def test_trees_of_many_units(hd):
    """256 nodes behind prefixes that end inside a page, at its end and nowhere."""
    c = ref.Case(4, 2, hd, [256, 200, 129], [37, 64, 0], seed=26)
    rng = np.random.default_rng(6)
    masks = np.concatenate([ref.masks_of(ref.random_parents(rng, n), 4) for n in (256, 200, 129)])
    _check(c, "tree", _call(c, "tree", masks, 4), masks)


@pytest.mark.parametrize("hd", [32, 128])
def test_thousands_of_sequences(hd):
    rng = np.random.default_rng(8)
    rows = [int(x) for x in rng.integers(0, 3, 2500)]
    past = [int(x) for x in rng.integers(0, 20, 2500)]
    c = ref.Case(2, 1, hd, rows, past, seed=27)
    _check(c, "packed", _call(c, "packed"))


class _Bound:
    """A call's device buffers, for running it many times."""

    def __init__(self, c):
        self.c = c
        self.q, k, v, table = dev(c.q), dev(c.k), dev(c.v), dev(c.table)
        self.start, self.past = dev(c.start), dev(np.array(c.past, np.int32))
        self.cache = ab.KvCache(k, v, table, c.stride, c.n_pages, c.KV, c.hd)
        self.out, self.ws = empty_f32(c.T * c.H * c.hd), _workspace()

    def run(self, stream):
        c = self.c
        ab.attention_packed(self.q, self.cache, self.start, self.past, len(c.past), c.T, c.H, c.scale, self.out, self.ws,
                            stream=stream)

    def check(self):
        c = self.c
        want, tol = ref.attention("packed", c.q, c.k, c.v, c.table, c.start, c.past, c.H, c.scale)
        assert np.all(np.abs(host(self.out).reshape(c.T, -1) - want) <= tol)


def _bound_pair():
    return (_Bound(ref.Case(8, 2, 128, [150, 9], [3, 500], seed=28)), _Bound(ref.Case(6, 6, 48, [200, 31], [0, 100], seed=29)),
            _Bound(ref.Case(8, 2, 128, [90, 1], [64, 1000], seed=30)))


def test_calls_at_once_on_several_streams():
    import torch
    calls = _bound_pair()
    streams = [torch.cuda.Stream() for _ in calls]
    torch.cuda.synchronize()
    for _ in range(8):
        for b, st in zip(calls, streams):
            b.run(st.cuda_stream)
    ab.device_sync()
    for b in calls:
        b.check()


def test_captured_calls_at_once():
    """Graphs with a workspace each, replayed on streams of their own."""
    import torch
    calls = _bound_pair()
    streams = [torch.cuda.Stream() for _ in calls]
    graphs = []
    torch.cuda.synchronize()
    for b, st in zip(calls, streams):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.stream(st):
            g.capture_begin()
            b.run(st.cuda_stream)
            b.run(st.cuda_stream)  # twice on one workspace, one behind the other
            g.capture_end()
        graphs.append(g)
    for _ in range(6):
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
    ab.device_sync()
    for b in calls:
        b.check()


FIRST_CALLS = """
import sys
sys.path[:0] = {paths!r}
import numpy as np, torch
import aaedn_b200 as ab, batched_ops_ref as ref
from gpu_util import dev, host
what = sys.argv[1]
st, g = torch.cuda.Stream(), torch.cuda.CUDAGraph()
s = st.cuda_stream
if what.startswith("attention"):
    c = ref.Case(4, 2, int(what[9:]), [70, 3], [5, 200], seed=31)
    q, cache = dev(c.q), ab.KvCache(dev(c.k), dev(c.v), dev(c.table), c.stride, c.n_pages, c.KV, c.hd)
    start, past, out = dev(c.start), dev(np.array(c.past, np.int32)), torch.zeros(c.T, c.H * c.hd, device="cuda")
    ws = torch.zeros(ab.ATTN_ROWS_WORKSPACE_BYTES, dtype=torch.uint8, device="cuda")
    call = lambda: ab.attention_packed(q, cache, start, past, 2, c.T, c.H, c.scale, out, ws, stream=s)
    want, tol = ref.attention("packed", c.q, c.k, c.v, c.table, c.start, c.past, c.H, c.scale)
    good = lambda: np.all(np.abs(host(out) - want) <= tol)
elif what == "pages":
    pool = torch.arange(4 * 64 * 8, dtype=torch.float32, device="cuda").view(4, 1, 64, 8)
    want = host(pool).copy()
    want[3] = want[1]
    want[3, :, 5] = want[3, :, 9]
    i = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")
    a1, a3, table, base, keep, ks = i(1), i(3), i(3), i(5), i(4), i(0, 1)
    def call():
        ab.kv_copy_pages([pool], 64 * 8, 4, a1, a3, 1, stream=s)
        ab.kv_compact([pool], 4, 1, 8, table, 1, base, keep, ks, 1, 1, stream=s)
    good = lambda: np.array_equal(host(pool), want)
else:
    rng = np.random.default_rng(3)
    lg, u = rng.normal(0, 2, (3, 5000)).astype(np.float32), rng.random(3).astype(np.float32)
    dl, du, tok = dev(lg), dev(u), torch.zeros(3, dtype=torch.int32, device="cuda")
    call = lambda: ab.sample_rows(dl, 3, 5000, None, None, None, None, du, tok, stream=s)
    good = lambda: list(host(tok)) == [ref.sample(lg[i], 1.0, 0, 1.0, 0.0, u[i]) for i in range(3)]
torch.cuda.synchronize()
with torch.cuda.stream(st):
    g.capture_begin()
    call()
    g.capture_end()
    g.replay()
ab.device_sync()
assert good(), what
print("good")
"""


@pytest.mark.parametrize("what", ["attention48", "attention128", "attention160", "pages", "sample"])
def test_the_first_call_of_a_process_can_be_captured(what):
    import os
    import subprocess
    import sys
    here = os.path.dirname(os.path.abspath(__file__))
    paths = [here, os.path.dirname(os.path.dirname(os.path.abspath(ab.__file__)))]
    r = subprocess.run([sys.executable, "-c", FIRST_CALLS.format(paths=paths), what], capture_output=True, text=True,
                       timeout=300)
    assert r.returncode == 0 and "good" in r.stdout, r.stdout + r.stderr


@pytest.mark.parametrize("hd", [132, 256])
def test_wide_heads(hd):
    """The cases above on the kernel for head_dim above 128."""
    test_infinities_and_nan_reach_the_rows_that_attend_them_only(hd)
    test_pages_outside_the_pool_and_slots_behind_the_table_are_left_out(hd)
    test_values_of_any_size(hd)
    test_thousands_of_sequences(hd)


def test_wide_heads_with_index_arrays_that_make_no_sense():
    import torch
    c = ref.Case(4, 2, 136, [20, 20], [64, 10], seed=32, poison=False)
    for start, past in (([0, 30, 20], [64, 10]), ([5, 10, 4000], [-7, -100]), ([-3, 8, 40], [2**31 - 1, 5]),
                        ([40, 20, 0], [0, 0]), ([2**31 - 1, -2**31, 7], [1, 1]), ([9, -2**31, 2**31 - 1], [3, 3])):
        out = torch.full((40, c.H * c.hd), 7.0, device="cuda")
        cache = ab.KvCache(dev(c.k), dev(c.v), dev(c.table), c.stride, c.n_pages, c.KV, c.hd)
        ab.attention_packed(dev(c.q), cache, dev(np.array(start, np.int32)), dev(np.array(past, np.int32)), 2, 40, c.H,
                            c.scale, out, _workspace())
        ab.device_sync()


def test_offsets_past_32_bits():
    """Pages whose byte and element offsets need more than 32 bits."""
    import torch
    KV, hd = 8, 128
    page = KV * 64 * hd
    n_pages = 2**32 // page + 40
    if torch.cuda.mem_get_info()[0] < 30 << 30:
        pytest.skip("needs 30 GB of free device memory")
    pool = torch.empty(n_pages * page, device="cuda")
    c = ref.Case(16, KV, hd, [70, 3], [50, 129], seed=24, spare=0, poison=False)
    far = n_pages - 1 - np.arange(c.n_pages)  # the last pages of the pool
    pv = pool.view(n_pages, KV, 64, hd)
    pv[torch.from_numpy(far.copy()).cuda()] = dev(c.k)
    table = np.where(c.table >= 0, far[c.table], -1).astype(np.int32)
    cache = ab.KvCache(pool, pool, dev(table), c.stride, n_pages, KV, hd)
    out = empty_f32(c.T * 16 * hd)
    ab.attention_packed(dev(c.q), cache, dev(c.start), dev(np.array(c.past, np.int32)), 2, c.T, 16, c.scale, out,
                        _workspace())
    ab.device_sync()
    got = host(out).reshape(c.T, -1)
    want, tol = ref.attention("packed", c.q, c.k, c.k, c.table, c.start, c.past, 16, c.scale)
    assert np.all(np.abs(got - want) <= tol)
    # the page operators on the same pool
    src, dst = dev(far[:2].astype(np.int32)), dev(np.array([0, int(far[2])], np.int32))
    ab.kv_copy_pages([pool], page, n_pages, src, dst, 2)
    torch.cuda.synchronize()
    assert torch.equal(pv[0], pv[int(far[0])]) and torch.equal(pv[int(far[2])], pv[int(far[1])])


def test_refuses_host_memory_and_a_small_workspace():
    c = ref.Case(4, 2, 64, [3], [0], seed=25)
    cache = ab.KvCache(dev(c.k), dev(c.v), dev(c.table), c.stride, c.n_pages, c.KV, c.hd)
    out, start, past = empty_f32(c.T * 256), dev(c.start), dev(np.array(c.past, np.int32))
    with pytest.raises(ab.AaednError) as e:
        ab.attention_packed(np.zeros((3, 256), np.float32).ctypes.data & ~15, cache, start, past, 1, 3, 4, 0.1, out,
                            _workspace())
    assert e.value.rc == ab.EINVAL and "device memory" in str(e.value)
    with pytest.raises(ab.AaednError) as e:
        ab.attention_packed(dev(c.q), cache, start, past, 1, 3, 4, 0.1, out, _workspace(), 1000)
    assert e.value.rc == ab.EINVAL and "workspace" in str(e.value)


# ------------------------------------------------------------- page operators
@pytest.mark.parametrize("arrays,pages,floats,pairs", [(1, 4, 4, 1), (3, 9, 64 * 3 * 32, 4), (64, 8, 8192, 3), (300, 5, 1028, 2)])
def test_copy_pages(arrays, pages, floats, pairs):
    rng = np.random.default_rng(floats)
    pools = [rng.normal(0, 1, (pages, floats)).astype(np.float32) for _ in range(arrays)]
    pick = rng.permutation(pages)[: 2 * pairs].astype(np.int32)
    src, dst = pick[:pairs], pick[pairs:]
    d = [dev(p) for p in pools]
    # pairs outside the pool, and a page onto itself, change nothing
    src2 = np.concatenate([src, [-1, pages, src[0], 0]]).astype(np.int32)
    dst2 = np.concatenate([dst, [dst[0], dst[0], src[0], pages + 3]]).astype(np.int32)
    ab.kv_copy_pages(d, floats, pages, dev(src2), dev(dst2), src2.size)
    for p, t in zip(pools, d):
        p[dst] = p[src]
        assert np.array_equal(host(t), p)


@pytest.mark.parametrize("arrays,KV,hd", [(2, 2, 128), (5, 3, 48), (260, 1, 4), (2, 8, 256)])
def test_compact(arrays, KV, hd):
    rng = np.random.default_rng(hd)
    S, pages, stride = 5, 20, 4
    table = rng.permutation(pages).reshape(S, stride).astype(np.int32)
    table[4, 2] = -1  # a page that is not there
    base = np.array([0, 63, 64, 150, 100], np.int32)
    keeps = [[0, 1, 2], [], [3, 4, 7, 9, 20, 21, 22, 23, 24, 40, 63], [5], [2, 3, 40, 50, 80]]
    start = np.concatenate([[0], np.cumsum([len(x) for x in keeps])]).astype(np.int32)
    flat = np.array([x for y in keeps for x in y], np.int32)
    pools = [rng.normal(0, 1, (pages, KV, 64, hd)).astype(np.float32) for _ in range(arrays)]
    d = [dev(p) for p in pools]
    ab.kv_compact(d, pages, KV, hd, dev(table), stride, dev(base), dev(flat), dev(start), S, flat.size)
    for p, t in zip(pools, d):
        for s in range(S):
            for i, j in enumerate(keeps[s]):
                a, b = base[s] + j, base[s] + i
                if max(a, b) >= stride * 64 or table[s, a // 64] < 0 or table[s, b // 64] < 0:
                    continue
                p[table[s, b // 64], :, b % 64] = p[table[s, a // 64], :, a % 64]
        assert np.array_equal(host(t), p)


def test_copy_more_pairs_than_a_grid_has_rows():
    import torch
    n = 70001
    pool = torch.arange(2 * n * 4, dtype=torch.float32, device="cuda").view(2 * n, 4)
    want = torch.cat([pool[:n], pool[:n].flip(0)])
    dst = torch.arange(2 * n - 1, n - 1, -1, dtype=torch.int32, device="cuda")
    ab.kv_copy_pages([pool], 4, 2 * n, torch.arange(n, dtype=torch.int32, device="cuda"), dst, n)
    assert torch.equal(pool, want)


def test_compaction_lists_that_make_no_sense_stay_in_bounds():
    """Descending list ends, negative and far slots: the pool's other pages stay."""
    rng = np.random.default_rng(9)
    host_pool = rng.normal(0, 1, (6, 2, 64, 8)).astype(np.float32)
    for start, keep, base in (([0, 3, 1], [5, -9, 2**31 - 1], [0, 10]), ([2, -2**31, 2**31 - 1], [1, 2, 3], [-5, 60]),
                              ([-4, 2, 900], [2**31 - 1, -2**31, 0], [2**31 - 1, -2**31])):
        d = dev(host_pool)
        ab.kv_compact([d], 6, 2, 8, dev(np.array([[1], [2]], np.int32)), 1, dev(np.array(base, np.int32)),
                      dev(np.array(keep, np.int32)), dev(np.array(start, np.int32)), 2, 3)
        ab.device_sync()
        assert np.array_equal(host(d)[[0, 3, 4, 5]], host_pool[[0, 3, 4, 5]])


# ------------------------------------------------------------------- sampling
def _sample(logits, T, k, p, m, u, ld=None):
    import torch
    B, V = logits.shape
    ld = ld or V
    lg = np.full((B, ld), 1e30, np.float32)
    lg[:, :V] = logits
    tok = torch.full((B + 1,), -5, dtype=torch.int32, device="cuda")
    arr = [None if x is None else dev(np.asarray(x, t)) for x, t in
           ((T, np.float32), (k, np.int32), (p, np.float32), (m, np.float32), (u, np.float32))]
    ab.sample_rows(dev(lg), B, V, *arr, tok, ld=ld)
    got = host(tok)
    assert got[B] == -5
    return got[:B]


def _want(logits, T, k, p, m, u):
    B = logits.shape[0]
    one = lambda x, d, i: d if x is None else x[i]  # noqa: E731
    return [ref.sample(logits[i], one(T, 1.0, i), one(k, 0, i), one(p, 1.0, i), one(m, 0.0, i), u[i]) for i in range(B)]


def _params(rng, B):
    return (rng.choice([0.0, 0.3, 0.7, 1.0, 1.5, 4.0], B), rng.choice([0, 1, 2, 40, 1000, -3, 10**9], B),
            rng.choice([1.0, 0.99, 0.9, 0.5, 0.01, 0.0, 2.0], B), rng.choice([0.0, 0.01, 0.3, 1.0, -1.0, 5.0], B),
            (rng.random(B) * (1 - 2.0 ** -24)).astype(np.float32))


@pytest.mark.parametrize("B,V", [(1, 1), (3, 2), (7, 31), (40, 1000), (5, 1025), (2, 8192), (4, 32000), (200, 4097),
                                 (3, 50257), (33, 128256), (2, 262145), (2, 300007)])
def test_sample_rows(B, V):
    rng = np.random.default_rng(B + V)
    lg = rng.normal(0, 3, (B, V)).astype(np.float32)
    lg[np.arange(B), rng.integers(0, V, B)] += rng.uniform(0, 12, B).astype(np.float32)
    prm = _params(rng, B)
    assert np.array_equal(_sample(lg, *prm), _want(lg, *prm))
    only_u = (None, None, None, None, prm[4])
    assert np.array_equal(_sample(lg, *only_u, ld=V + 3), _want(lg, *only_u))


@pytest.mark.parametrize("V", [1000, 40000, 128256])
def test_sample_rows_with_ties(V):
    """Logits on a coarse grid, all equal, and two values: order by id."""
    rng = np.random.default_rng(V)
    B = 48
    lg = (rng.integers(-6, 7, (B, V)) * 0.5).astype(np.float32)
    lg[:8] = 1.25
    lg[8:16] = np.where(rng.random((8, V)) < 0.5, np.float32(-3.0), np.float32(-3.0000002))
    lg[16:20] = np.where(rng.random((4, V)) < 0.5, np.float32(0.0), np.float32(-0.0))
    prm = _params(rng, B)
    prm[4][:4] = (0.0, 0.5, 0.25, 1 - 2.0 ** -24)
    assert np.array_equal(_sample(lg, *prm), _want(lg, *prm))


def test_sample_rows_with_infinities_and_nan():
    rng = np.random.default_rng(9)
    B, V = 24, 5000
    lg = rng.normal(0, 2, (B, V)).astype(np.float32)
    lg[0:4, 10:] = -np.inf
    lg[4:8][rng.random((4, V)) < 0.3] = np.nan
    lg[8] = np.nan
    lg[9] = -np.inf
    lg[10, [7, 9]] = np.inf
    lg[11:14, ::2] = -1e30
    lg[14:16] = np.float32(-3.4e38)
    lg[14:16, 100] = 3.4e38
    lg[16:18, 5:] = np.float32(np.finfo(np.float32).min)
    T, k, p, m, u = _params(rng, B)
    T = np.where(T == 0, 1.0, T)
    assert np.array_equal(_sample(lg, T, k, p, m, u), _want(lg, T, k, p, m, u))
    assert np.array_equal(_sample(lg, np.full(B, np.nan), k, p, m, u), _want(lg, np.zeros(B), k, p, m, u))


def test_sample_rows_draws_the_distribution_of_its_uniforms():
    """Every u of a fine grid: each token's share is its probability to a step."""
    V, N = 12, 4096
    lg = np.random.default_rng(3).normal(0, 1, V).astype(np.float32)
    u = ((np.arange(N) + 0.5) / N).astype(np.float32)
    got = _sample(np.tile(lg, (N, 1)), None, None, None, None, u)
    p = np.exp(lg.astype(np.float64))
    p /= p.sum()
    assert np.all(np.abs(np.bincount(got, minlength=V) / N - p) <= 1.0 / N + 1e-9)


def test_sample_rows_agrees_with_the_one_row_sampler():
    rng = np.random.default_rng(6)
    lg = rng.normal(0, 2, (1, 3001)).astype(np.float32)
    for u in (0.03, 0.3, 0.9):
        tok = dev(np.zeros(1, np.uint32).view(np.int32))
        ab.sample(dev(lg), 3001, 0.8, 0.9, u, tok)
        assert _sample(lg, [0.8], None, [0.9], None, [u])[0] == host(tok)[0]


@pytest.mark.parametrize("B,V", [(620, 3001), (300, 50257), (150, 128256), (76, 190001)])
def test_sample_more_rows_than_the_gpu_holds(B, V):
    """Several rounds of CTAs, for rows of one CTA and of more."""
    rng = np.random.default_rng(B)
    lg = rng.normal(0, 2, (B, V)).astype(np.float32)
    lg[np.arange(B), rng.integers(0, V, B)] += rng.uniform(0, 9, B).astype(np.float32)
    prm = _params(rng, B)
    got, want = _sample(lg, *prm), _want(lg, *prm)
    assert np.array_equal(got, want), np.argwhere(got != np.array(want))[:5]


@pytest.mark.parametrize("V", [900, 5000, 40001])
@pytest.mark.parametrize("k", [3, 300, 700, 1500, 2048, 2049, 4000])
@pytest.mark.parametrize("spread,shift", [(2, 0), (0.001, 7.3), (80, 0), (3, -200)])
def test_sample_top_k_of_any_size(V, k, spread, shift):
    """Lists that are short, long and too long, of logits of any range."""
    rng = np.random.default_rng(V + k)
    lg = (rng.normal(0, spread, (4, V)) + shift).astype(np.float32)
    T = [spread, 0.5 * spread, 2.0 * spread, 1.0]
    p, m, u = [1.0, 0.9, 0.7, 1.0], [0.0, 0.0, 0.0, 0.01], rng.random(4).astype(np.float32) * np.float32(1 - 2.0 ** -24)
    got, want = _sample(lg, T, [k] * 4, p, m, u), _want(lg, T, [k] * 4, p, m, u)
    assert np.array_equal(got, want)


@pytest.mark.parametrize("T", [float("inf"), 1e38, 1e-30, 1e-44])
def test_sample_temperatures_at_the_ends(T):
    rng = np.random.default_rng(10)
    lg = rng.integers(-3, 4, (6, 3000)).astype(np.float32)
    lg[:, ::7] = -np.inf
    u = rng.random(6).astype(np.float32)
    for k in (0, 100):
        got, want = _sample(lg, [T] * 6, [k] * 6, None, None, u), _want(lg, [T] * 6, [k] * 6, None, None, u)
        assert np.array_equal(got, want)


def test_sample_rows_captured():
    import torch
    rng = np.random.default_rng(7)
    lg = rng.normal(0, 2, (6, 9000)).astype(np.float32)
    d, tok = dev(lg), torch.zeros(6, dtype=torch.int32, device="cuda")
    u = dev(rng.random(6).astype(np.float32))
    st = torch.cuda.Stream()
    g = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.stream(st):
        g.capture_begin()
        ab.sample_rows(d, 6, 9000, None, None, None, None, u, tok, stream=st.cuda_stream)
        g.capture_end()
    for seed in (1, 2):
        nu = np.random.default_rng(seed).random(6).astype(np.float32)
        u.copy_(torch.from_numpy(nu))
        g.replay()
        assert np.array_equal(host(tok), _want(lg, None, None, None, None, nu))
