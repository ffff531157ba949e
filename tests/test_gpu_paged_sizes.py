"""The operators over a paged cache at the ends of their ranges: the most sequences, many
without rows, more of them than are split into parts, single tokens beside chunks, more
KV heads than the chip has places, pages that several texts share, rows that are written
past the L2s, captures without a workspace."""
import ctypes as C

import numpy as np
import pytest

import edgecore_amd as ec
from test_gpu_paged_ops import append_case, attn_case, call, check, check_append, check_edit, check_read, edit_case, half, random_pages, rows_of
from test_gpu_tree_ops import _Graph

pytestmark = pytest.mark.gpu

MOST = 65535


def many_case(seed, type, KVH, hd, past, new):
    """More sequences than texts: ten of these, which they share."""
    past, new = np.asarray(past), np.asarray(new)
    c = attn_case(seed, type, KVH, KVH, hd, 16, [int((past + new).max())] * 10, [0] * 10, pad=0)
    c["pages"].table = c["pages"].table[np.arange(len(past)) % 10]
    M = int(new.sum()) + 3
    return {**c, "past": past.astype(np.int32), "new": new.astype(np.int32),
            "start": np.concatenate(([0], np.cumsum(new))).astype(np.int32),
            "q": np.random.default_rng(seed).normal(0, 1, (M, KVH * hd)).astype(np.float32)}


def test_attention_of_the_most_sequences():
    r = np.random.default_rng(1)
    past = r.integers(0, 4, MOST)
    c = attn_case(1, "int8", 2, 1, 16, 4, past, [1] * MOST)
    at = [0, 1, 15, 16, 17, 32767, 50000, MOST - 1]
    got = check(c, rows=[(b, 0) for b in at])
    assert np.isfinite(got[:MOST]).all()


@pytest.mark.parametrize("KVH", [1, 12])
def test_attention_of_few_among_the_most_sequences(KVH):
    new = np.zeros(MOST, int)
    new[[0, 40000, MOST - 1]] = [2, 1, 19]
    past = np.full(MOST, 1)
    c = attn_case(2, "fp16", 2 * KVH, KVH, 16, 4, past, new)
    check(c)


def test_appends_of_the_most_sequences():
    r = np.random.default_rng(3)
    c = append_case(3, "int8", 2, 1, 16, 4, r.integers(0, 4, MOST), [1] * MOST)
    q, pages = ec.paged_append_dev(c["pages"], c["qkv"], 2, c["past"], c["start"])
    x = c["qkv"][:MOST].reshape(MOST, 4, 16)
    assert np.array_equal(q[:MOST], c["qkv"][:MOST, :32])
    page, at = pages.table[:, 0], c["past"]
    for n, i in (("k", 2), ("v", 3)):
        codes, s = getattr(pages, n)[page, 0, at].view(np.int8), half(getattr(pages, n + "_scale")[page, 0, at])
        # codes are steps of a scale that is within a step of fp16 above max / 127
        y = x[:, i].astype(np.float64)
        top = np.abs(y).max(-1)
        assert (s >= top / 127).all() and (s <= top / 127 * (1 + 2.0 ** -10)).all()
        assert np.array_equal(codes, np.rint(y / s[:, None]))


def test_reads_of_the_most_sequences():
    r = np.random.default_rng(4)
    pages = random_pages(r, "fp16", 1, 16, 4, [4] * MOST)
    count = r.integers(0, 5, MOST)
    z = np.full((MOST, 4, 16), 0x1234, np.uint16)
    got = ec.paged_read_dev(pages, z, z, [0] * MOST, count)
    for n, g in zip(("k", "v"), got):
        want = np.where((np.arange(4) < count[:, None])[..., None], getattr(pages, n)[pages.table[:, 0], 0], 0x1234)
        assert np.array_equal(g, want)


def test_edits_of_the_most_rows():
    r = np.random.default_rng(5)
    for B, N in ((MOST, 1), (1, MOST)):
        c = dict(logits=r.normal(0, 3, (B * N, 5)).astype(np.float32), N=N, text=r.integers(0, 5, (B, 3)).astype(np.int32),
                 len=r.integers(0, 4, B).astype(np.int32), presence=r.uniform(0, 1, B).astype(np.float32))
        got = ec.logits_edit_dev(**c)
        has = ((c["text"][..., None] == np.arange(5)) & (np.arange(3)[:, None] < c["len"][:, None, None])).any(1)
        want = c["logits"] - np.where(has, c["presence"][:, None], 0).astype(np.float32).repeat(N, 0)
        assert np.array_equal(got, want)


@pytest.mark.parametrize("type,hd", [("int8", 64), ("fp16", 128)])
def test_attention_of_many_sequences_unsplit(type, hd):
    """More sequences and KV heads than are split: single tokens over longer texts; tiles of
    16 rows of sequences with more; chunks."""
    r = np.random.default_rng(6)
    past = r.integers(0, 1500, 200)
    past[[3, 150]] = [1500, 0]
    c = many_case(6, type, 12, hd, past, [1] * 200)
    check(c, rows=[(b, 0) for b in (0, 3, 4, 150, 199)])
    check(c, 100, 4, rows=[(b, 0) for b in (0, 3, 4, 150, 199)])
    new = r.integers(0, 3, 250)
    new[[0, 100, 249]] = [0, 77, 33]
    c = many_case(7, type, 12, hd, r.integers(0, 300, 250), new)
    check(c, rows=[(100, 0), (100, 15), (100, 16), (100, 76), (101, 0), (249, 0), (249, 32)])
    new = r.integers(0, 200, 110)
    new[[0, 50, 109]] = [130, 0, 257]
    c = many_case(8, type, 12, hd, r.integers(0, 100, 110), new)
    check(c, rows=[(0, 0), (0, 127), (0, 128), (0, 129), (49, 0), (51, 0), (109, 0), (109, 128), (109, 256)])
    check(c, 40, 2, rows=[(0, 0), (0, 128), (0, 129), (109, 0), (109, 127), (109, 256)])


@pytest.mark.parametrize("type", ec.CACHE_TYPES)
@pytest.mark.parametrize("H,KVH,hd", [(14, 2, 64), (12, 2, 128), (16, 4, 96), (3, 1, 16)])
def test_attention_of_single_tokens_beside_a_chunk(type, H, KVH, hd):
    """Sequences of up to 16 rows of a KV head, and of one more, among tiles of 128."""
    G = H // KVH
    r = np.random.default_rng(hd)
    new = [16 // G, 1, 333, 16 // G + 1, 0] + [1] * 19
    past = np.concatenate(([3000, 0, 1500, 700, 5], r.integers(0, 2000, 19)))
    c = attn_case(hd, type, H, KVH, hd, 32, past, new)
    rows = [(0, i) for i in range(new[0])] + [(3, i) for i in range(new[3])] + [(1, 0), (2, 0), (2, 127), (2, 332), (7, 0), (23, 0)]
    check(c, rows=rows)
    check(c, 200, 4, rows=rows)
    check(c, 64, 0, rows=rows)


@pytest.mark.parametrize("KVH,G", [(600, 1), (513, 2)])
@pytest.mark.parametrize("new", [[1, 1], [140, 3]])
def test_attention_of_more_heads_than_places(KVH, G, new):
    check(attn_case(9, "int8", KVH * G, KVH, 16, 16, [200, 90], new), rows=[(0, 0), (0, new[0] - 1), (1, new[1] - 1)])


@pytest.mark.parametrize("type", ["fp16", "e4m3"])
@pytest.mark.parametrize("new", [[1, 1, 1], [60, 20, 33]])
def test_shared_prefix(type, new):
    """Texts whose first pages are the same ones: as with pages of their own that hold the same."""
    c = attn_case(10, type, 12, 2, 128, 16, [700, 640, 900], new)
    own = c["pages"]
    for b in (1, 2):
        for n in ("k", "v") + (() if type == "fp16" else ("k_scale", "v_scale")):
            a = getattr(own, n)
            a[own.table[b, :40]] = a[own.table[0, :40]]
    want = check(c)
    c["pages"].table[1:, :40] = c["pages"].table[0, :40]
    assert np.array_equal(call(c), want)
    z = np.zeros((3, 700, 256), np.uint16)
    k, v = ec.paged_read_dev(own, z, z, [0, 0, 0], [640] * 3)
    for name, g in (("k", k), ("v", v)):
        assert np.array_equal(half(g[2, :640]), rows_of(own, name, 0, 640).reshape(640, 256)) and np.array_equal(g[1, :640], g[0, :640])


def test_rows_past_the_l2s():
    """Outputs larger than the L2s: the same as in smaller calls."""
    c = edit_case(11, 10, 7, 151936, 300, 20, True)
    c["nodes"][1:4] = [0, 7, 3]
    got = ec.logits_edit_dev(**c)
    odd = {**c, "logits": np.ascontiguousarray(c["logits"][:, :151935])}
    odd_got = ec.logits_edit_dev(**odd)
    for b in range(10):
        rows = slice(7 * b, 7 * b + 7)
        part = {n: a if n == "N" else a[rows] if n in ("logits", "mask") else a[b:b + 1] for n, a in c.items()}
        want = ec.logits_edit_dev(**part)
        assert np.array_equal(got[rows], want) and np.array_equal(odd_got[rows], want[:, :151935])
    check_edit({n: a if n == "N" else a[:7] if n in ("logits", "mask") else a[:1] for n, a in c.items()})
    for type in ec.CACHE_TYPES:
        pages = random_pages(np.random.default_rng(12), type, 2, 128, 64, [6000] * 6)
        check_read(pages, [0, 1, 2, 3, 64, 6000], [6000, 5000, 5998, 0, 5936, 0], 6, 6100, None, [0, 9, 102, 0, 64, 0])


def test_appends_of_other_widths():
    """Rows of heads that leave a wave's last lanes, and a block's last waves, without one."""
    for H, KVH, hd, rot in ((1, 1, 4, 0), (3, 3, 12, 8), (7, 1, 36, 32), (5, 5, 100, 96), (2, 1, 132, 128), (1, 1, 256, 256)):
        for layout in (0, 1):
            c = append_case(hd, "int8", H, KVH, hd, 16, [0, 40], [5, 1])
            c["qg"], c["kg"] = None, np.random.default_rng(1).normal(1, 0.2, hd).astype(np.float32)
            check_append(c, ec.rope_inv_freq(rot, 1e4) if rot else None, layout)


def test_capture_without_a_workspace():
    """A captured call whose workspace is not there yet is refused, the capture ends as ever,
    and the same call runs after an eager one has made it."""
    L = ec.lib()
    if L.ec_release():
        pytest.skip("models are loaded")
    c = attn_case(13, "int8", 12, 2, 128, 16, [3000, 100], [1, 1], pad=0)
    E = 12 * 128
    with ec._Call() as k:
        cache = c["pages"].put(k)
        a = [C.byref(cache), k.put("q", c["q"], np.float32), E, 12, None, k.put("past", c["past"], np.int32), 2, 2, 3000, 0, 0,
             k.put("out", np.full_like(c["q"], 7.25), np.float32), E]
        read = lambda: k.get("out", np.float32, c["q"].shape)  # noqa: E731
        run = lambda: L.ec_attention_paged_dev(*a)  # noqa: E731
        with pytest.raises(AssertionError, match="inside a stream capture"):
            _Graph(run)
        assert (read() == 7.25).all()
        assert run() == 0 and L.ec_sync() == 0
        want = read()
        g = _Graph(run)
        for _ in range(3):
            g.replay()
            assert L.ec_sync() == 0 and np.array_equal(read(), want)
        # a larger call moves the workspace; the graph keeps its own
        check(attn_case(14, "fp16", 12, 2, 128, 16, [9000, 8000], [300, 200]), rows=[(0, 299), (1, 0)])
        for _ in range(3):
            g.replay()
            assert L.ec_sync() == 0 and np.array_equal(read(), want)
        g.close()
        check(c, got=np.concatenate((want, np.full((1, E), 7.25, np.float32))))


@pytest.mark.parametrize("type", ec.CACHE_TYPES)
@pytest.mark.parametrize("H,KVH,hd", [(12, 2, 128), (16, 4, 96), (14, 2, 64), (8, 1, 32)])
def test_chunks_same_bits(type, H, KVH, hd):
    """Every result is there when it is read: equal calls give equal bits."""
    c = attn_case(17, type, H, KVH, hd, 16, [3000], [500])
    want = check(c, rows=[(0, 0), (0, 300), (0, 499)])
    for _ in range(8):
        assert np.array_equal(call(c), want)


def test_same_call_same_bits():
    """Nothing depends on an order of arrival."""
    for args in (("e4m3", 14, 2, 64, 64, [7500, 100], [200, 1]), ("int8", 12, 2, 128, 16, [4000, 30, 900], [1, 1, 1])):
        c = attn_case(15, *args)
        want = call(c)
        for _ in range(3):
            assert np.array_equal(call(c), want)
    e = edit_case(16, 4, 8, 5000, 3000, 40, True, few=50)
    want = ec.logits_edit_dev(**e)
    for _ in range(3):
        assert np.array_equal(ec.logits_edit_dev(**e), want)
