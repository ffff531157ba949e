"""The operators over a paged cache (quantised appends, attention of new tokens,
rows read back) and the edits of logits against plain 64-bit implementations, at the
sizes, masks and values where they can go wrong.

Tolerances are worst-case bounds of the 32-bit arithmetic, written where they
are used; whole numbers, codes' steps and copied rows are equal."""
import ctypes as C
import math

import numpy as np
import pytest

import edgecore_amd as ec
from test_gpu_tree_ops import _Graph, f16, lineage, ref_sample, trees

pytestmark = pytest.mark.gpu

U = 2.0 ** -24  # half a step of fp32
NAN16, INF16 = 0x7E00, 0x7C00
TYPES = ec.CACHE_TYPES


def e4m3_table():
    c = np.arange(256)
    e, m = (c >> 3) & 15, c & 7
    v = np.where(e > 0, (8 + m) * 2.0 ** (e - 10.0), m * 2.0 ** -9)
    v[(c & 127) == 127] = np.nan
    return np.where(c >= 128, -v, v)


E4M3 = e4m3_table()


def half(bits):
    return bits.view(np.float16).astype(np.float64)


def values(pages, name):
    """[npages][KVH][page][hd]: what the rows stand for, in 64 bits."""
    a, s = getattr(pages, name), getattr(pages, name + "_scale")
    if pages.type == "fp16":
        return half(a)
    codes = a.view(np.int8).astype(np.float64) if pages.type == "int8" else E4M3[a]
    with np.errstate(over="ignore", invalid="ignore"):
        return (codes * half(s)[..., None]).astype(np.float16).astype(np.float64)


def random_pages(rng, type, KVH, hd, page, rows):
    """A cache with room for `rows` rows of each sequence, pages in any order, some of
    nobody's."""
    B = len(rows)
    per = max(1, max(-(-r // page) for r in rows))
    npages = B * per + 2
    table = rng.permutation(npages)[:B * per].reshape(B, per).astype(np.int32)
    shape = (npages, KVH, page, hd)
    if type == "fp16":
        return ec.Pages(type, f16(rng.normal(0, 1, shape)), f16(rng.normal(0, 1, shape)), table)
    kv = []
    for _ in range(2):
        if type == "int8":
            kv.append(np.clip(np.rint(rng.normal(0, 42, shape)), -127, 127).astype(np.int8).view(np.uint8))
        else:
            c = rng.integers(0, 256, shape)
            kv.append(np.where((c & 127) >= 0x70, c & 0x8F, c).astype(np.uint8))  # up to 120
    s = [f16(np.exp(rng.normal(0, 0.3, shape[:3])) / (42 if type == "int8" else 30)) for _ in range(2)]
    return ec.Pages(type, kv[0], kv[1], table, *s)


def rows_of(pages, name, b, n):
    """The first n rows of sequence b's text, [n][KVH][hd]."""
    page = pages.k.shape[2]
    p = np.arange(n)
    return values(pages, name)[pages.table[b, p // page], :, p % page]


# ---------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------

def attn_case(seed, type, H, KVH, hd, page, past, new, pad=3):
    rng = np.random.default_rng(seed)
    past, new = np.array(past, np.int32), np.array(new, np.int32)
    M = int(new.sum()) + pad
    return dict(H=H, past=past, new=new, start=np.concatenate(([0], np.cumsum(new))).astype(np.int32),
                pages=random_pages(rng, type, KVH, hd, page, past + new), q=rng.normal(0, 1, (M, H * hd)).astype(np.float32))


def call(c, window=0, sinks=0, **k):
    return ec.attention_paged_dev(c["pages"], c["q"], c["H"], c["past"], c["start"], window, sinks,
                                  out=np.full_like(c["q"], 7.25), **k)


def sees(t, window, sinks):
    p = np.arange(t + 1)
    return p[(p > t - window) | (p < sinks)] if window else p


def check(c, window=0, sinks=0, rows=None, got=None, **k):
    """Every row (or those of `rows`, (sequence, row) each) against 64 bits."""
    H, pages = c["H"], c["pages"]
    _, KVH, _, hd = pages.k.shape
    G = H // KVH
    if got is None:
        got = call(c, window, sinks, **k)
    assert (got[c["start"][-1]:] == 7.25).all()  # padding is as it was
    se = sw = 0.0
    for b in range(len(c["past"])):
        which = [i for i in range(c["new"][b]) if rows is None or (b, i) in rows]
        if not which:
            continue
        n = int(c["past"][b] + c["new"][b])
        kk, vv = (rows_of(pages, m, b, n) for m in ("k", "v"))
        for i in which:
            at = sees(int(c["past"][b]) + i, window, sinks)
            q = c["q"][c["start"][b] + i].astype(np.float64).reshape(KVH, G, hd)
            ka, va = kk[at].transpose(1, 2, 0), vv[at].transpose(1, 0, 2)
            x = q @ ka / math.sqrt(hd)
            size = np.abs(q) @ np.abs(ka) / math.sqrt(hd)
            p = np.exp(x - x.max(-1, keepdims=True))
            p /= p.sum(-1, keepdims=True)
            want = p @ va
            # a score is off by the roundings of its hd + 2 steps and of its q (2^-22 where
            # it is split in two 16-bit parts), a weight by twice that and its own
            # exponential's, the sum by one rounding a term
            dx = size * (hd + 8) * 2 * U + np.abs(x) * 4 * U
            tol = (p * (2 * dx.max(-1, keepdims=True) + (len(at) + 16) * 2 * U)) @ np.abs(va) + 1e-30
            err = np.abs(got[c["start"][b] + i].reshape(want.shape) - want)
            assert (err <= tol).all(), (b, i, err.max(), (err / tol).max())
            se, sw = se + (err ** 2).sum(), sw + (want ** 2).sum()
    if sw:
        # independent roundings of hd + n terms (with 8 for chance): what a 16-bit
        # rounding of q or of the weights would pass 10 times over
        span = hd + int((c["past"] + c["new"]).max())
        assert math.sqrt(se / sw) <= 8 * U * math.sqrt(span), math.sqrt(se / sw)
    return got


HEADS = [(14, 2, 64), (12, 2, 128), (12, 12, 64), (16, 4, 96), (8, 1, 32), (10, 5, 80), (4, 2, 112), (3, 1, 16), (3, 3, 20),
         (2, 1, 250), (5, 1, 7), (2, 2, 512)]


@pytest.mark.parametrize("type", TYPES)
@pytest.mark.parametrize("H,KVH,hd", HEADS)
@pytest.mark.parametrize("page,past,new", [(16, [0, 1, 63, 64, 65, 130, 700], [1] * 7), (24, [0, 31, 200], [5, 1, 17]),
                                           (64, [190, 0, 7], [33, 64, 3]), (7, [0, 129], [130, 70])])
def test_attention_heads(type, H, KVH, hd, page, past, new):
    check(attn_case(hd * page + H, type, H, KVH, hd, page, past, new))


@pytest.mark.parametrize("type,H,KVH,hd", [("int8", 14, 2, 64), ("fp16", 12, 12, 64), ("e4m3", 12, 2, 128), ("int8", 3, 3, 20)])
@pytest.mark.parametrize("new", [[1, 1, 1, 1], [70, 1, 40, 9]])
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (2, 4), (7, 0), (64, 4), (100, 64), (333, 65), (333, 5000), (5000, 4),
                                          (2147483647, 2147483647), (64, 2147483647)])
def test_attention_window(type, H, KVH, hd, new, window, sinks):
    check(attn_case(window % 1000 + sinks % 100, type, H, KVH, hd, 16, [0, 3, 97, 700], new), window, sinks)


@pytest.mark.parametrize("type", TYPES)
@pytest.mark.parametrize("H,KVH,hd", [(14, 2, 64), (12, 2, 128), (5, 1, 7)])
def test_attention_ragged(type, H, KVH, hd):
    """Sequences without rows, first, last and between; many of one row beside a chunk."""
    check(attn_case(5, type, H, KVH, hd, 16, [20, 0, 77, 300, 64, 9], [0, 3, 0, 150, 1, 0]))
    c = attn_case(6, type, H, KVH, hd, 16, [7 * b % 331 for b in range(90)], [1] * 40 + [200] + [1] * 49)
    check(c, rows=[(0, 0), (39, 0), (40, 0), (40, 199), (41, 0), (89, 0)])
    check(c, 50, 2, rows=[(0, 0), (39, 0), (40, 0), (40, 100), (41, 0), (89, 0)])


@pytest.mark.parametrize("type", TYPES)
def test_attention_without_starts(type):
    """A row each: the same as with starts."""
    c = attn_case(7, type, 14, 2, 64, 16, [0, 5, 99, 640], [1] * 4, pad=0)
    want = check(c)
    got = ec.attention_paged_dev(c["pages"], c["q"], 14, c["past"], out=np.full_like(c["q"], 7.25))
    assert np.array_equal(got, want)


@pytest.mark.parametrize("type,H,KVH,hd,page,past,new,rows", [
    ("fp16", 14, 2, 64, 16, [32000], [64], [(0, 0), (0, 31), (0, 63)]),
    ("int8", 12, 2, 128, 16, [9000, 3001], [1, 1], None),
    ("e4m3", 12, 2, 128, 64, [4000, 100], [300, 40], [(0, 0), (0, 150), (0, 299), (1, 3), (1, 39)]),
    ("int8", 12, 12, 64, 32, [1000 - 7 * b for b in range(16)], [1] * 16, None),
    ("fp16", 12, 2, 128, 32, [0, 0], [1500, 700], [(0, 0), (0, 1), (0, 63), (0, 64), (0, 777), (0, 1499), (1, 0), (1, 699)]),
    ("e4m3", 2, 1, 250, 16, [5000], [3], None),
])
def test_attention_long(type, H, KVH, hd, page, past, new, rows):
    check(attn_case(len(past) + new[0], type, H, KVH, hd, page, past, new), rows=rows)


@pytest.mark.parametrize("type", TYPES)
@pytest.mark.parametrize("H,KVH,hd", [(14, 2, 64), (12, 2, 128), (16, 4, 96), (5, 1, 7)])
@pytest.mark.parametrize("new", [[1, 1], [100, 9]])
def test_attention_unseen_values(type, H, KVH, hd, new):
    """NaN and infinities in rows that a token does not see (behind its own, in front of
    the window, other pages) do not reach it; in rows that it sees they do."""
    c = attn_case(21, type, H, KVH, hd, 16, [150, 90], new)
    pages = c["pages"]
    clean = check(c)
    page = 16
    n = c["past"] + c["new"]
    at = lambda b, p: (pages.table[b, p // page], slice(None), p % page)  # noqa: E731

    def spoil(name, where, bad):
        # 8-bit rows: by their scale
        a = getattr(pages, name) if type == "fp16" else getattr(pages, name + "_scale")
        kept = a[where].copy()
        a[where] = bad
        return lambda: a.__setitem__(where, kept)

    # pages of nobody, and what is behind the texts in their last pages
    for name in ("k", "v"):
        for p in set(range(pages.k.shape[0])) - set(pages.table.ravel()):
            spoil(name, (p,), NAN16)
        for b in range(2):
            for p in range(n[b], pages.table.shape[1] * page):
                spoil(name, at(b, p), INF16 if p % 2 else NAN16)
    assert np.array_equal(call(c), clean)
    # one row of the text and the chunk's own rows: those that do not see it keep their values
    for p in (40, 149, 150, int(n[0]) - 1):
        for name, bad in (("v", NAN16), ("v", INF16), ("k", NAN16), ("k", INF16)):
            undo = spoil(name, at(0, p), bad)
            for window, sinks in ((0, 0), (30, 0), (30, 41)):
                was = clean if not window else call_clean(c, window, sinks, undo, lambda: spoil(name, at(0, p), bad))
                got = call(c, window, sinks)
                for i in range(c["new"][0]):
                    if p in sees(150 + i, window, sinks):
                        assert not np.isfinite(got[i]).all() or name == "k", (p, name, i)
                    else:
                        assert np.allclose(got[i], was[i], rtol=0, atol=1e-5), (p, name, i, window)
                assert np.array_equal(got[c["new"][0]:], was[c["new"][0]:])
            undo()


def call_clean(c, window, sinks, undo, again):
    undo()
    got = call(c, window, sinks)
    again()
    return got


@pytest.mark.parametrize("H,KVH,hd", [(14, 2, 64), (12, 2, 128), (8, 1, 32), (5, 1, 7)])
@pytest.mark.parametrize("new", [[1, 1], [90, 5]])
def test_attention_seen_values(H, KVH, hd, new):
    """One element of an fp16 value that is not finite: the outputs of that element and its
    KV head are not finite, all others are as they were; of a key: the KV head's."""
    c = attn_case(22, "fp16", H, KVH, hd, 16, [700, 90], new)
    clean = check(c, rows=[(0, 0), (1, 0)])
    pages, n0 = c["pages"], new[0]
    for p in (300, 700):
        at = (pages.table[0, p // 16], KVH - 1, p % 16, hd // 2)
        for a, bad in ((pages.v, NAN16), (pages.v, INF16), (pages.k, NAN16)):
            kept = a[at]
            a[at] = bad
            got = call(c)
            a[at] = kept
            hit = np.zeros((len(got), KVH, H // KVH, hd), bool)
            if a is pages.v:
                hit[:n0, -1, :, hd // 2] = True
            else:
                hit[:n0, -1] = True
            hit = hit.reshape(len(got), H * hd)
            assert not np.isfinite(got[hit]).any() and np.array_equal(got[~hit], clean[~hit])


def peaked(seed, type, H, KVH, hd, past, new, at, gap, size=1.0, mixed=False):
    """Keys of which one, at place `at` of the text, points where the queries do: its
    score stands about gap above the sum of the others' weights (and values with a mean)."""
    c = attn_case(seed, type, H, KVH, hd, 16, past, new)
    rng, pages = np.random.default_rng(seed + 1), c["pages"]
    d = rng.choice([-1.0, 1.0], (KVH, hd))
    q = rng.normal(0, 1, (len(c["q"]), H, hd)) + np.repeat(d, H // KVH, 0)
    if mixed:
        q[:, 1::2] -= 2 * np.repeat(d, H // KVH, 0)[1::2]
    c["q"] = (q * size).reshape(len(q), H * hd).astype(np.float32)
    for b, n in enumerate(past):
        p = min(int(at * n), n - 1)
        k = d * (math.log(n) + 1.0 + gap) / math.sqrt(hd)
        pg, o = pages.table[b, p // 16], p % 16
        if type == "fp16":
            pages.k[pg, :, o] = f16(k)
            pages.v[pg, :, o] = f16(rng.normal(0, 0.02, k.shape))
        else:
            one = 127 if type == "int8" else 0x7E  # 448
            sign = np.where(d > 0, one, 256 - one if type == "int8" else one | 0x80)
            pages.k[pg, :, o] = sign
            pages.k_scale[pg, :, o] = f16(np.abs(k[:, 0]) / (127 if type == "int8" else 448))
    if size != 1.0:  # the keys as much larger or smaller
        if type == "fp16":
            with np.errstate(over="ignore"):
                pages.k[...] = f16(half(pages.k) / size)
        else:
            pages.k_scale[...] = f16(half(pages.k_scale) / size)
    return c


def check_peaked(c, rows, window=0, sinks=0):
    """Root mean squares of the errors over the rows' elements: at most four times plain
    fp32's (numpy) and 2^-20 of the outputs'.  (The score of a position that takes a share s
    of the weight is some 20 in units of log2, and half a step of it 2^-20: each of its sums,
    4 to 8, is off by that, independently, in all by 2^-18 for the largest heads; it moves
    the output by s (1 - s) <= 1/4 of what lies between the values.)"""
    H, pages = c["H"], c["pages"]
    _, KVH, _, hd = pages.k.shape
    got = call(c, window, sinks)
    err = plain = size = 0.0

    def attend(q, k, v, dt):
        x = (q.astype(dt) @ k.astype(dt).transpose(1, 2, 0)) * dt(1 / math.sqrt(hd))
        w = np.exp(x - x.max(-1, keepdims=True))
        return (w @ v.astype(dt).transpose(1, 0, 2)) / w.sum(-1, keepdims=True, dtype=dt)

    for b, i in rows:
        n = int(c["past"][b]) + i
        at = sees(n, window, sinks)
        k, v = (rows_of(pages, m, b, n + 1)[at] for m in ("k", "v"))
        q = c["q"][c["start"][b] + i].reshape(KVH, H // KVH, hd)
        want, f32 = attend(q, k, v, np.float64), attend(q, k, v, np.float32)
        err += ((got[c["start"][b] + i].reshape(want.shape) - want) ** 2).sum()
        plain += ((f32 - want) ** 2).sum()
        size += (want ** 2).sum()
    err, plain, size = (math.sqrt(x) for x in (err, plain, size))
    print("error %.2e, plain fp32 %.2e of the outputs" % (err / size, plain / size))
    assert err <= 4 * plain + 2.0 ** -20 * size, (err / size, plain / size)


SHAPES = [(14, 2, 64), (12, 2, 128), (16, 4, 96), (8, 1, 32), (5, 1, 40)]


@pytest.mark.parametrize("type", TYPES)
@pytest.mark.parametrize("H,KVH,hd", SHAPES)
@pytest.mark.parametrize("past,new", [([1000, 1000], [1, 1]), ([4000, 1000], [90, 20])])
@pytest.mark.parametrize("gap", [0.0, 2.0, 4.6])
def test_first_token_takes_most(type, H, KVH, hd, past, new, gap):
    """Shares of about 1/2, 0.9 and 0.99."""
    check_peaked(peaked(int(10 * gap) + new[0], type, H, KVH, hd, past, new, 0.0, gap), [(0, 0), (1, new[1] - 1)])


@pytest.mark.parametrize("type,H,KVH,hd,new", [("fp16", 14, 2, 64, 64), ("int8", 12, 2, 128, 1), ("e4m3", 14, 2, 64, 200)])
@pytest.mark.parametrize("gap", [0.0, 4.6])
def test_first_token_of_a_long_text(type, H, KVH, hd, new, gap):
    check_peaked(peaked(int(10 * gap) + new, type, H, KVH, hd, [32000], [new], 0.0, gap), [(0, 0), (0, new - 1)])


@pytest.mark.parametrize("type,H,KVH,hd", [("fp16", 14, 2, 64), ("int8", 12, 2, 128), ("e4m3", 12, 12, 64), ("int8", 5, 1, 40)])
@pytest.mark.parametrize("new", [[1, 1], [60, 60]])
@pytest.mark.parametrize("at", [0.0, 0.5, 0.97, 1.0])
@pytest.mark.parametrize("gap", [-3.0, 5.0, 20.0])
@pytest.mark.parametrize("mixed", [False, True])
def test_maximum_that_moves(type, H, KVH, hd, new, at, gap, mixed):
    """The position with the largest score in the first tile, the middle, the last tiles,
    up to 30 above what came before; of all rows of a wave, or of every second one."""
    check_peaked(peaked(new[0], type, H, KVH, hd, [1500, 1499], new, at, gap, mixed=mixed), [(0, 0), (1, new[1] - 1)])


@pytest.mark.parametrize("type,H,KVH,hd", [("fp16", 14, 2, 64), ("fp16", 12, 2, 128), ("int8", 8, 1, 32)])
@pytest.mark.parametrize("new", [[1, 1], [40, 9]])
@pytest.mark.parametrize("size", [2.0 ** -9, 64.0, 2.0 ** 13])
def test_sizes_of_queries(type, H, KVH, hd, new, size):
    if type == "int8" and size > 100:
        size = 2.0 ** 5  # fp16 scales end at 2^-24
    check_peaked(peaked(7, type, H, KVH, hd, [700, 650], new, 0.6, 3.0, size=size, mixed=True), [(0, 0), (1, new[1] - 1)])


@pytest.mark.parametrize("H,KVH,hd", [(14, 2, 64), (12, 2, 128)])
@pytest.mark.parametrize("new", [[9], [40]])
def test_rows_of_unlike_sizes(H, KVH, hd, new):
    """Rows of one wave from 2^-40 to 2^17."""
    c = peaked(9, "fp16", H, KVH, hd, [900], new, 0.4, 3.0)
    n = len(c["q"]) * H
    c["q"] = (c["q"].reshape(n, hd) * 2.0 ** np.resize([0, -40, 17, 0, -9, 2, 5], n).reshape(n, 1)).reshape(-1, H * hd).astype(np.float32)
    check_peaked(c, [(0, i) for i in range(0, new[0], 3)])


@pytest.mark.parametrize("window,sinks", [(500, 1), (1200, 0)])
def test_first_token_as_a_sink(window, sinks):
    for H, KVH, hd in ((14, 2, 64), (12, 2, 128)):
        for new in ([1], [70]):
            for at in (0.0, 1.0 - window / 2500, 1.0 - (window - 4) / 2500):
                check_peaked(peaked(window, "int8", H, KVH, hd, [2500], new, at, 4.6), [(0, 0), (0, new[0] - 1)], window, sinks)


@pytest.mark.parametrize("H,KVH,hd", [(14, 2, 64), (12, 2, 128), (5, 1, 40)])
@pytest.mark.parametrize("new", [[1, 1], [40, 3]])
def test_infinite_queries(H, KVH, hd, new):
    """NaN in its own row and head alone."""
    c = attn_case(11, "int8", H, KVH, hd, 16, [703, 40], new)
    clean = call(c).reshape(-1, H, hd)
    for bad in (np.inf, -np.inf, np.nan):
        q = c["q"][0, hd + 1]
        c["q"][0, hd + 1] = bad
        got = call(c).reshape(-1, H, hd)
        c["q"][0, hd + 1] = q
        assert np.isnan(got[0, 1]).all()
        got[0, 1] = clean[0, 1]
        # (when a row's maximum moves decides when its neighbours' do, by their room)
        assert np.abs(got - clean).max() < 1e-5


BAD = [("past", 1, -1), ("past", 1, -2 ** 31), ("past", 1, 2 ** 31 - 1), ("past", 1, 1000), ("table", (1, 0), -1),
       ("table", (1, 1), 10 ** 6), ("table", (1, 0), 2 ** 31 - 1)]


@pytest.mark.parametrize("new", [[1, 1, 1], [40, 20, 33]])
@pytest.mark.parametrize("hd", [64, 20])
@pytest.mark.parametrize("name,at,value", BAD)
def test_attention_bad_numbers(hd, new, name, at, value):
    """A sequence whose numbers name no rows, or whose pages are none, is marked; the
    others are as ever."""
    c = attn_case(31, "int8", 4, 2, hd, 16, [50, 60, 40], new)
    clean = check(c)
    (c["pages"].table if name == "table" else c[name])[at] = value
    got = call(c)
    mine = slice(c["start"][1], c["start"][2])
    assert np.isnan(got[mine]).all()
    got[mine] = clean[mine]
    assert np.array_equal(got, clean)


@pytest.mark.parametrize("new", [[1, 1, 1], [40, 20, 33]])
def test_attention_pages_out_of_sight(new):
    """Entries of the table that no token of the call sees are not looked at."""
    c = attn_case(32, "e4m3", 4, 2, 64, 16, [500, 600, 400], new)
    clean = check(c, 100, 4)
    for b in range(3):
        c["pages"].table[b, 1:(int(c["past"][b]) - 100) // 16] = -5
        c["pages"].table[b, -(-int(c["past"][b] + c["new"][b]) // 16):] = 10 ** 9
    assert np.array_equal(call(c, 100, 4), clean)


@pytest.mark.parametrize("start", [[0, 5, 3, 8], [3, 2, 1, 0], [-7, 2, 2, 9], [0, 2 ** 31 - 1, 5, 9], [-2 ** 31, 2 ** 31 - 1, 0, 4],
                                   [2, 4, 4, 5], [0, 40, 41, 45], [9, 9, 9, 9], [0, 9, 0, 9]])
@pytest.mark.parametrize("hd", [64, 20])
def test_attention_odd_starts(hd, start):
    """Starts that do not ascend, or pass the rows: nothing is read or written out of
    place, and where they do ascend every row is right."""
    c = attn_case(33, "int8", 4, 2, hd, 16, [50, 60, 40], [3, 3, 3], pad=0)
    c["start"] = np.array(start, np.int32)
    got = call(c)
    ok = all(0 <= a <= b <= 9 for a, b in zip(start, start[1:]))
    if ok:
        c["new"] = np.diff(c["start"])
        assert (got[:start[0]] == 7.25).all()
        check(c, got=np.concatenate((got, np.full((1, 4 * hd), 7.25, np.float32))))


@pytest.mark.parametrize("new", [[1, 1], [50, 3]])
def test_attention_max_past(new):
    c = attn_case(34, "int8", 12, 2, 128, 16, [300, 200], new)
    want = check(c, max_past=300)
    got = call(c, max_past=299)
    assert np.isnan(got[:new[0]]).all() and np.array_equal(got[new[0]:], want[new[0]:])


@pytest.mark.parametrize("type", TYPES)
@pytest.mark.parametrize("H,KVH,hd", [(14, 2, 64), (12, 2, 128), (5, 1, 7)])
@pytest.mark.parametrize("new", [[1, 1], [60, 3]])
def test_attention_strides_and_alignment(type, H, KVH, hd, new):
    """Rows of q and out with a stride, 4 bytes off 16; the cache 2 bytes (codes: 1) off."""
    c = attn_case(41, type, H, KVH, hd, 16, [300, 77], new)
    pages, E, M = c["pages"], H * hd, len(c["q"])
    want = check(c)
    esz = 2 if type == "fp16" else 1
    for ldq, off, coff in ((E, 0, 0), (E + 4, 4, 0), (E + 3, 1, 0), (E, 0, esz)):
        with ec._Call() as k:
            qx = np.zeros((M + 1, ldq), np.float32)
            qx.ravel()[off:off + M * ldq].reshape(M, ldq)[:, :E] = c["q"]
            ox = np.full((M + 1) * ldq, 3.5, np.float32)
            q, o = k.put("q", qx, np.float32), k.put("o", ox, np.float32)
            cache = pages.put(k)
            if coff:
                for n in ("k", "v"):
                    raw = np.concatenate((np.zeros(coff, np.uint8), getattr(pages, n).view(np.uint8).ravel()))
                    setattr(cache, n, k.put(n + "x", raw, np.uint8) + coff)
            rc = ec.lib().ec_attention_paged_dev(C.byref(cache), q + 4 * off, ldq, H, k.put("start", c["start"], np.int32),
                                                 k.put("past", c["past"], np.int32), 2, M, 300, 0, 0, o + 4 * off, ldq)
            assert rc == 0, ec.last_error()
            assert ec.lib().ec_sync() == 0
            got = k.get("o", np.float32, (M + 1) * ldq)
        rows = got[off:off + M * ldq].reshape(M, ldq)
        assert (got[:off] == 3.5).all() and (got[off + M * ldq:] == 3.5).all() and (rows[:, E:] == 3.5).all()
        assert (rows[c["start"][-1]:] == 3.5).all()
        full = rows[:, :E].copy()
        full[c["start"][-1]:] = 7.25
        check(c, got=full)
        if not off % 4 and not coff:
            assert np.array_equal(full, want)


@pytest.mark.parametrize("H,KVH,hd", [(14, 2, 64), (5, 1, 7)])
@pytest.mark.parametrize("past,new", [([900, 40], [1, 1]), ([0, 40], [70, 9])])
def test_attention_in_place(H, KVH, hd, past, new):
    """out = q, in parts and without."""
    c = attn_case(42, "e4m3", H, KVH, hd, 16, past, new, pad=0)
    want = check(c)
    with ec._Call() as k:
        q, cache = k.put("q", c["q"], np.float32), c["pages"].put(k)
        rc = ec.lib().ec_attention_paged_dev(C.byref(cache), q, H * hd, H, k.put("start", c["start"], np.int32),
                                             k.put("past", c["past"], np.int32), 2, len(c["q"]), max(past), 0, 0, q, H * hd)
        assert rc == 0 and ec.lib().ec_sync() == 0
        assert np.array_equal(k.get("q", np.float32, c["q"].shape), want)


@pytest.mark.parametrize("type", ["fp16", "int8"])
@pytest.mark.parametrize("new", [1, 40])
def test_past_32_bits(type, new):
    """Pages that lie more than 2^32 bytes into the cache: written, attended, read back."""
    H, KVH, hd, page = 4, 2, 128, 64
    esz = 2 if type == "fp16" else 1
    npages = 2 ** 32 // (KVH * page * hd * esz) + 40
    c = attn_case(43, type, H, KVH, hd, page, [1000], [new], pad=0)
    pages, per = c["pages"], c["pages"].table.shape[1]
    L = ec.lib()
    far = (npages - 1 - np.arange(per)).astype(np.int32)
    size = KVH * page * hd * esz
    bufs = [ec.DeviceBuffer(npages * size) for _ in range(2)]
    scales = [ec.DeviceBuffer(npages * KVH * page * 2) for _ in range(2)]
    try:
        with ec._Call() as k:
            for i, p in enumerate(far):
                old = pages.table[0, i]
                for buf, sc, n in zip(bufs, scales, ("k", "v")):
                    a = np.ascontiguousarray(getattr(pages, n)[old])
                    assert L.ec_memcpy_h2d(buf.ptr + int(p) * size, a.ctypes.data, a.nbytes) == 0
                    if type != "fp16":
                        a = np.ascontiguousarray(getattr(pages, n + "_scale")[old])
                        assert L.ec_memcpy_h2d(sc.ptr + int(p) * KVH * page * 2, a.ctypes.data, a.nbytes) == 0
            cache = ec.PagedCache(bufs[0].ptr, bufs[1].ptr, scales[0].ptr, scales[1].ptr, TYPES.index(type), npages, page, KVH, hd,
                                  k.put("table", far[None], np.int32), per)
            start, past = k.put("start", c["start"], np.int32), k.put("past", c["past"], np.int32)
            q, out = k.put("q", c["q"], np.float32), k.put("out", np.zeros_like(c["q"]), np.float32)
            x = np.random.default_rng(3).normal(0, 1, (new, (H + 2 * KVH) * hd)).astype(np.float32)
            kc = [k.put(n, np.zeros((1, 1000 + new, KVH * hd), np.uint16), np.uint16) for n in ("kc", "vc")]
            rc = (L.ec_attention_paged_dev(C.byref(cache), q, H * hd, H, start, past, 1, new, 1000, 0, 0, out, H * hd)
                  or L.ec_paged_append_dev(C.byref(cache), k.put("x", x, np.float32), x.shape[1], q, H * hd, H, None, None, 0.0, None,
                                           0, 0, 1.0, start, past, 1, new)
                  or L.ec_paged_read_dev(C.byref(cache), k.put("first", [0], np.int32), k.put("count", [1000 + new], np.int32), 1,
                                         1000 + new, *kc, 1, 1000 + new, None, None))
            assert rc == 0 and L.ec_sync() == 0, ec.last_error()
            check(c, got=np.concatenate((k.get("out", np.float32, c["q"].shape), np.full((1, H * hd), 7.25, np.float32))))
            for n, first in (("k", H), ("v", H + KVH)):
                got = half(k.get(n + "c", np.uint16, (1000 + new, KVH, hd)))
                assert np.array_equal(got[:1000], rows_of(pages, n, 0, 1000))
                y = x.reshape(new, H + 2 * KVH, hd)[:, first:first + KVH].astype(np.float64)
                assert np.array_equal(got[1000:], store(y, type)[0])
    finally:
        for b in bufs + scales:
            b.close()


# ---------------------------------------------------------------------------
# append
# ---------------------------------------------------------------------------

def store(y, type):
    """(values, scales) that rows in 64 bits are stored as."""
    if type == "fp16":
        return y.astype(np.float16).astype(np.float64), None
    Q = 127.0 if type == "int8" else 448.0
    t = np.abs(y).max(-1, keepdims=True) / Q
    h = up16(t)
    z = y / np.where(h > 0, h, 1.0)
    if type == "int8":
        z = np.rint(z)
    else:
        e = np.maximum(np.floor(np.log2(np.maximum(np.abs(z), 2.0 ** -20))), -6)
        z = np.rint(z / 2.0 ** (e - 3)) * 2.0 ** (e - 3)
    return (np.clip(z, -Q, Q) * h).astype(np.float16).astype(np.float64), h[..., 0]


def up16(t):
    with np.errstate(over="ignore"):
        h = t.astype(np.float16)
    return np.where(h.astype(np.float64) < t, np.nextafter(h, np.float16(np.inf)), h).astype(np.float64)


def append_case(seed, type, H, KVH, hd, page, past, new, norm=True, pad=2):
    rng = np.random.default_rng(seed)
    past, new = np.array(past, np.int32), np.array(new, np.int32)
    M = int(new.sum()) + pad
    return dict(H=H, past=past, new=new, start=np.concatenate(([0], np.cumsum(new))).astype(np.int32),
                pages=random_pages(rng, type, KVH, hd, page, past + new),
                qkv=rng.normal(0, 3, (M, (H + 2 * KVH) * hd)).astype(np.float32),
                qg=rng.normal(1, 0.3, hd).astype(np.float32) if norm else None,
                kg=rng.normal(1, 0.3, hd).astype(np.float32) if norm else None)


def check_append(c, inv_freq=None, layout=0, factor=1.0, eps=1e-6, bad=()):
    H, pages = c["H"], c["pages"]
    _, KVH, page, hd = pages.k.shape
    M, type = len(c["qkv"]), pages.type
    q, after = ec.paged_append_dev(pages, c["qkv"], H, c["past"], c["start"], c["qg"], c["kg"], eps, inv_freq, layout, factor,
                                   np.full((M, H * hd), 7.25, np.float32))
    rot = 0 if inv_freq is None else 2 * len(inv_freq)
    assert (q[c["start"][-1]:] == 7.25).all()
    x = c["qkv"].astype(np.float64).reshape(M, H + 2 * KVH, hd)
    names = ("k", "v") + (() if type == "fp16" else ("k_scale", "v_scale"))
    want = {n: getattr(pages, n).copy() for n in names}
    for b in range(len(c["past"])):
        n, r = c["new"][b], slice(c["start"][b], c["start"][b + 1])
        if b in bad:
            assert np.isnan(q[r]).all()
            continue
        if not n:
            continue
        pos = c["past"][b] + np.arange(n)
        ang = pos[:, None].astype(np.float64) * (inv_freq if rot else np.zeros(0))
        y = {}
        for name, first, heads, gamma in (("q", 0, H, c["qg"]), ("k", H, KVH, c["kg"])):
            z = x[r, first:first + heads]
            if gamma is not None:
                z = z / np.sqrt((z ** 2).mean(-1, keepdims=True) + eps) * gamma
            z, w = z.copy(), z
            i0 = 2 * np.arange(rot // 2) if layout else np.arange(rot // 2)
            i1 = i0 + 1 if layout else i0 + rot // 2
            cs, sn = (factor * f(ang)[:, None, :] for f in (np.cos, np.sin))
            z[..., i0], z[..., i1] = w[..., i0] * cs - w[..., i1] * sn, w[..., i0] * sn + w[..., i1] * cs
            size = np.abs(w)
            size[..., i0] = size[..., i1] = (np.abs(w[..., i0]) + np.abs(w[..., i1])) * abs(factor)
            y[name] = z, size
        z, size = y["q"]
        # the norm: hd roundings in the sum (half of it in the root) and four more;
        # sine and cosine to two units; three roundings of the rotation
        err = np.abs(q[r].reshape(z.shape) - z)
        assert (err <= size * (hd / 2 + 14) * U + 1e-30).all(), (b, err.max())
        y["v"] = x[r, H + KVH:], np.abs(x[r, H + KVH:])
        at = (pages.table[b, pos // page], slice(None), pos % page)
        for name in ("k", "v"):
            z, size = y[name]
            # in 64 bits: positions up to 2^17 make angles of 2^17, off by 2^-36; a hundredth
            # of a millionth of the row's elements covers that and every other rounding
            slack = 1e-8 * size.max(-1, keepdims=True)
            got = values(after, name)[at]
            if type == "fp16":
                assert (np.abs(got - z) <= slack + np.maximum(np.abs(z) * 2.0 ** -11, 2.0 ** -25)).all(), (b, name)
            else:
                Q = 127.0 if type == "int8" else 448.0
                h = half(getattr(after, name + "_scale")[at])
                t = np.abs(z).max(-1) / Q
                assert ((h >= up16(np.maximum(t - slack[..., 0], 0))) & (h <= up16(t + slack[..., 0]))).all(), (b, name)
                a = getattr(after, name)[at]
                code = a.view(np.int8).astype(np.float64) if type == "int8" else E4M3[a]
                w = z / np.where(h > 0, h, 1.0)[..., None]
                step = 1.0 if type == "int8" else 2.0 ** (np.maximum(np.floor(np.log2(np.maximum(np.abs(w), 2.0 ** -20))), -6) - 3)
                # the nearest code
                room = slack / np.where(h > 0, h, 1.0)[..., None]
                assert (np.abs(code - w) <= step / 2 + room).all() and (np.abs(code) <= Q).all(), (b, name)
                if name == "v":
                    assert np.array_equal(got, store(z, type)[0])
                want[name + "_scale"][at] = getattr(after, name + "_scale")[at]
            want[name][at] = getattr(after, name)[at]
    for n in names:
        assert np.array_equal(getattr(after, n), want[n]), n  # nothing else was written
    return q, after


@pytest.mark.parametrize("type", TYPES)
@pytest.mark.parametrize("H,KVH,hd", [(14, 2, 64), (12, 2, 128), (12, 12, 64), (10, 5, 80), (16, 4, 96), (9, 3, 42), (3, 1, 256),
                                      (2, 2, 512), (2, 1, 7), (1, 1, 1), (1, 1, 4), (64, 8, 128)])
@pytest.mark.parametrize("layout", [0, 1])
def test_append_heads(type, H, KVH, hd, layout):
    for past, new, norm in (([0, 5, 70], [1, 1, 1], True), ([3, 0, 40], [7, 20, 1], False)):
        c = append_case(hd + new[0], type, H, KVH, hd, 16, past, new, norm)
        check_append(c)
        for rot in {hd // 2 * 2, hd // 4 * 2, hd // 8 * 8, 2}:
            if 0 < rot <= hd:
                check_append(c, ec.rope_inv_freq(rot, 1e4), layout)


@pytest.mark.parametrize("kind,factor", [(0, 1.0), (1, 1.1), (2, 1.0), (3, 1.0)])
def test_append_far_positions(kind, factor):
    check_append(append_case(3, "int8", 4, 2, 64, 128, [32000, 131070, 60001], [2, 2, 2]), ec.rope_inv_freq(64, 1e4, kind, 8.0, 4096.0),
                 0, factor)


@pytest.mark.parametrize("type", TYPES)
@pytest.mark.parametrize("page", [1, 3, 16, 24, 1000])
def test_append_pages(type, page):
    """Pages of any size, sequences without rows."""
    check_append(append_case(4, type, 6, 2, 64, page, [10, 0, 300, 64, 7], [33, 0, 1, 90, 0]), ec.rope_inv_freq(64, 1e6))


@pytest.mark.parametrize("type", TYPES)
@pytest.mark.parametrize("hd", [64, 42])
def test_append_values(type, hd):
    """Rows of zeros, tiny and large ones, of one outlier, of ties; NaN and infinities."""
    c = append_case(11, type, 2, 2, hd, 16, [9], [9], norm=False)
    x = c["qkv"].reshape(-1, 6, hd)
    x[0] = 0.0
    x[1] *= 1e-7
    x[2] *= 3000.0
    x[3] = 0.001
    x[3, :, 3] = 60000.0
    x[4] = (np.arange(hd) % 20 - 10) * 0.5
    x[4, :, 0] = 127.0  # a scale of 1: halves of a code
    x[5] = (np.arange(hd) % 30 - 15) * 0.0625
    x[5, :, 0] = 448.0
    x[6, :, 0] = 2.0 ** -24
    x[7] = -65000.0
    check_append(c)
    for bad in (np.nan, np.inf, -np.inf):
        x[8, 3, 5] = bad  # the second key
        _, after = ec.paged_append_dev(c["pages"], c["qkv"], 2, c["past"], c["start"])
        got = values(after, "k")[c["pages"].table[0, 17 // 16], :, 17 % 16]
        assert np.isfinite(got[0]).all()
        assert not np.isfinite(got[1, 5]) and (type == "fp16" or np.isnan(got[1]).all())


@pytest.mark.parametrize("type", TYPES)
@pytest.mark.parametrize("hd", [64, 42])
def test_append_in_place(type, hd):
    """q the first columns of qkv."""
    c = append_case(12, type, 14, 2, hd, 16, [9, 0], [5, 30], pad=0)
    inv = ec.rope_inv_freq(hd, 1e4)
    want, after = check_append(c, inv)
    M, W = c["qkv"].shape
    with ec._Call() as k:
        x, cache = k.put("x", c["qkv"], np.float32), c["pages"].put(k)
        rc = ec.lib().ec_paged_append_dev(C.byref(cache), x, W, x, W, 14, k.put("qg", c["qg"], np.float32),
                                          k.put("kg", c["kg"], np.float32), 1e-6, k.put("f", inv, np.float64), hd, 0, 1.0,
                                          k.put("start", c["start"], np.int32), k.put("past", c["past"], np.int32), 2, M)
        assert rc == 0 and ec.lib().ec_sync() == 0
        got = k.get("x", np.float32, (M, W))
        assert np.array_equal(got[:, :14 * hd], want) and np.array_equal(got[:, 14 * hd:], c["qkv"][:, 14 * hd:])
        a = c["pages"].got(k)
        assert np.array_equal(a.k, after.k) and np.array_equal(a.v, after.v)


@pytest.mark.parametrize("name,at,value", BAD[:4] + [("table", (1, 3), -1), ("table", (1, 3), 10 ** 6)])
@pytest.mark.parametrize("hd", [64, 42])
def test_append_bad_numbers(hd, name, at, value):
    c = append_case(13, "int8", 4, 2, hd, 16, [50, 60, 40], [2, 3, 5])
    (c["pages"].table if name == "table" else c[name])[at] = value
    check_append(c, bad=(1,))


def test_append_one_bad_page():
    """Of a sequence's rows those on a page outside the cache are marked."""
    c = append_case(14, "e4m3", 4, 2, 64, 16, [10, 0], [40, 2])
    want, after = check_append(c)
    bad = int(c["pages"].table[0, 1])
    c["pages"].table[0, 1] = -1
    q, got = ec.paged_append_dev(c["pages"], c["qkv"], 4, c["past"], c["start"], c["qg"], c["kg"], q=np.full_like(want, 7.25))
    assert np.isnan(q[6:22]).all()
    q[6:22] = want[6:22]
    assert np.array_equal(q, want)
    keep = [p for p in range(after.k.shape[0]) if p != bad]
    assert np.array_equal(got.k[keep], after.k[keep])


@pytest.mark.parametrize("start", [[0, 5, 3, 8], [3, 2, 1, 0], [-7, 2, 2, 9], [0, 2 ** 31 - 1, 5, 9], [2, 4, 4, 5], [0, 40, 41, 45]])
def test_append_odd_starts(start):
    c = append_case(15, "int8", 2, 1, 64, 16, [5, 6, 4], [3, 3, 3], pad=0)
    c["start"] = np.array(start, np.int32)
    if all(0 <= a <= b <= 9 for a, b in zip(start, start[1:])):
        c["new"] = np.diff(c["start"])
        q, _ = ec.paged_append_dev(c["pages"], c["qkv"], 2, c["past"], c["start"], q=np.full((9, 128), 7.25, np.float32))
        assert (q[:start[0]] == 7.25).all() and (q[start[-1]:] == 7.25).all()
        c["qg"] = c["kg"] = None
        check_append(c)
    else:
        ec.paged_append_dev(c["pages"], c["qkv"], 2, c["past"], c["start"])


# ---------------------------------------------------------------------------
# read back
# ---------------------------------------------------------------------------

def check_read(pages, first, count, nslots, Cr, slot=None, to=None, skip=(), **k):
    _, KVH, _, hd = pages.k.shape
    rng = np.random.default_rng(1)
    cache = [f16(rng.normal(0, 1, (nslots, Cr, KVH * hd))) for _ in range(2)]
    got = ec.paged_read_dev(pages, *cache, first, count, slot, to, **k)
    for name, g, want in zip(("k", "v"), got, cache):
        for b in range(len(first)):
            if b in skip:
                continue
            s, t = b if slot is None else slot[b], 0 if to is None else to[b]
            y = rows_of(pages, name, b, first[b] + count[b])[first[b]:]
            want[s, t:t + count[b]] = y.astype(np.float16).view(np.uint16).reshape(-1, KVH * hd)
        assert np.array_equal(g, want)


@pytest.mark.parametrize("type", TYPES)
@pytest.mark.parametrize("KVH,hd", [(2, 64), (2, 128), (12, 64), (5, 80), (3, 20), (1, 7), (2, 512)])
@pytest.mark.parametrize("page", [16, 24, 7])
def test_read(type, KVH, hd, page):
    rng = np.random.default_rng(hd)
    pages = random_pages(rng, type, KVH, hd, page, [200, 17, 90, 1])
    check_read(pages, [0, 0, 0, 0], [200, 17, 90, 1], 4, 200)
    check_read(pages, [3, 16, 90, 0], [150, 1, 0, 1], 6, 300, [5, 0, 1, 3], [0, 299, 300, 7])
    check_read(pages, [3, 16, 50, 0], [15, 1, 20, 1], 1, 300, [0, 0, 0, 0], [0, 15, 16, 299], max_count=40)


@pytest.mark.parametrize("arg,value", [(0, -1), (0, 2 ** 31 - 1), (0, 10 ** 6), (1, -1), (1, 41), (1, 2 ** 31 - 1), (2, -1), (2, 3),
                                       (3, -1), (3, 280), (3, 2 ** 31 - 1)])
def test_read_bad_numbers(arg, value):
    pages = random_pages(np.random.default_rng(5), "int8", 2, 64, 16, [90, 90, 90])
    a = [[5, 6, 7], [30, 40, 20], [2, 0, 1], [0, 10, 20]]
    a[arg][1] = value
    check_read(pages, a[0], a[1], 3, 300, a[2], a[3], skip=(1,), max_count=40)


def test_read_same_rows_twice():
    """The first of two sequences whose rows of a slot overlap is read, whatever its order."""
    pages = random_pages(np.random.default_rng(6), "e4m3", 2, 64, 16, [90] * 70)
    slot, to = np.arange(70), np.zeros(70, int)
    slot[69], to[69] = 3, 29
    slot[40], to[40] = 39, 30  # beside it
    check_read(pages, [0] * 70, [30] * 70, 70, 100, slot, to, skip=(69,))


def test_read_bad_page():
    pages = random_pages(np.random.default_rng(7), "fp16", 2, 64, 16, [90, 90])
    kept = pages.table[0, 2]
    pages.table[0, 2] = -1
    z = np.zeros((2, 90, 128), np.uint16)
    k, v = ec.paged_read_dev(pages, z, z, [0, 0], [90, 90])
    pages.table[0, 2] = kept
    for name, g in (("k", k), ("v", v)):
        assert np.isnan(half(g[0, 32:48])).all()
        want = np.stack([rows_of(pages, name, b, 90).reshape(90, 128) for b in range(2)])
        want[0, 32:48] = np.nan
        assert np.array_equal(half(g), want, equal_nan=True)


# ---------------------------------------------------------------------------
# logits
# ---------------------------------------------------------------------------

def edit_case(seed, B, N, V, T, bias=0, mask=False, token=True, few=None):
    r = np.random.default_rng(seed)
    c = dict(logits=r.normal(0, 3, (B * N, V)).astype(np.float32), N=N,
             text=r.integers(0, few or V, (B, T)).astype(np.int32), len=r.integers(0, T + 1, B).astype(np.int32))
    c["prompt"] = (c["len"] * r.random(B)).astype(np.int32)
    c["repetition"] = r.uniform(0.7, 1.5, B).astype(np.float32)
    c["frequency"], c["presence"] = (r.uniform(-0.5, 1.0, B).astype(np.float32) for _ in range(2))
    if token:
        c["token"], c["parent"] = r.integers(0, few or V, (B, N)).astype(np.int32), trees(r, B, N)
    if N > 1:
        c["nodes"] = r.integers(0, N + 1, B).astype(np.int32)
        c["nodes"][0] = N
    if bias:
        c["bias_token"], c["bias"] = r.integers(0, few or V, (B, bias)).astype(np.int32), r.normal(0, 5, (B, bias)).astype(np.float32)
        c["nbias"] = r.integers(0, bias + 1, B).astype(np.int32)
    if mask:
        c["mask"] = r.integers(0, 2 ** 32, (B * N, (V + 31) // 32 + 2), dtype=np.uint32)
        c["mask"][0] = 0
    return c


def check_edit(c, bad=(), got=None):
    """fp32 throughout: at most four roundings, of numbers no larger than `size`."""
    x, N = c["logits"], c["N"]
    B, V = len(x) // N, x.shape[1]
    out = np.full_like(x, 7.25)
    if got is None:
        got = ec.logits_edit_dev(**c, out=out)
    g = lambda n, b, d: d if c.get(n) is None else c[n][b]  # noqa: E731
    for b in range(B):
        n = int(g("nodes", b, N))
        if b in bad:
            n = n if 0 <= n <= N else N
            assert np.isnan(got[b * N:b * N + n]).all() and (got[b * N + n:(b + 1) * N] == 7.25).all()
            continue
        assert (got[b * N + n:(b + 1) * N] == 7.25).all()
        lines = lineage(list(c["parent"][b]) if c.get("parent") is not None else range(-1, N - 1))
        for i in range(n):
            text = [] if c.get("text") is None else list(c["text"][b, :c["len"][b]])
            p = min(max(int(g("prompt", b, 0)), 0), len(text))
            after = text[p:] + ([] if c.get("token") is None else [c["token"][b, j] for j in lines[i]])
            count = np.zeros(V)
            for t in after:
                if 0 <= t < V:
                    count[t] += 1
            seen = count > 0
            seen[[t for t in text if 0 <= t < V]] = True
            y = x[b * N + i].astype(np.float64)
            rep = float(g("repetition", b, 1.0))
            y = np.where(seen, np.where(y > 0, y / rep, y * rep), y)
            size = np.abs(y) + count * abs(float(g("frequency", b, 0))) + abs(float(g("presence", b, 0)))
            y = y - np.where(count > 0, float(g("frequency", b, 0)) * count + float(g("presence", b, 0)), 0.0)
            if c.get("bias") is not None:
                last = {}
                for k in range(int(g("nbias", b, c["bias"].shape[1]))):
                    last[int(c["bias_token"][b, k])] = float(c["bias"][b, k])
                for t, v in last.items():
                    if 0 <= t < V:
                        y[t] += v
                        size[t] += abs(v)
            if c.get("mask") is not None:
                y[np.unpackbits(c["mask"][b * N + i].view(np.uint8), bitorder="little")[:V] == 0] = -np.inf
            row = got[b * N + i].astype(np.float64)
            assert np.array_equal(np.isneginf(row), np.isneginf(y))
            f = np.isfinite(y)
            assert (np.abs(row[f] - y[f]) <= 5 * U * size[f]).all(), (b, i)
            same = f & ~seen
            if c.get("bias") is not None:
                same[[t for t in last if 0 <= t < V]] = False
            assert np.array_equal(row[same], x[b * N + i].astype(np.float64)[same])
    return got


@pytest.mark.parametrize("V", [1, 2, 31, 32, 33, 255, 1000, 4095, 4096, 4097, 50257, 151936])
def test_edit_sizes(V):
    few = min(V, 40)
    check_edit(edit_case(V, 3, 1, V, 50, token=False, few=few))
    check_edit(edit_case(V + 1, 2, 5, V, 50, bias=7, mask=True, few=few))


@pytest.mark.parametrize("B,N,T,bias,mask", [(1, 1, 1, 0, False), (1, 64, 3000, 0, True), (9, 3, 70, 300, False), (40, 1, 500, 3, True),
                                             (2, 17, 9000, 1000, True)])
def test_edit_batches(B, N, T, bias, mask):
    check_edit(edit_case(B + N, B, N, 5000, T, bias, mask))
    check_edit(edit_case(B + N + 1, B, N, 5000, T, bias, mask, few=20))


def test_edit_parts():
    """Every argument alone, and none."""
    full = edit_case(5, 3, 4, 700, 40, 9, True, few=60)
    base = dict(logits=full["logits"], N=4)
    assert np.array_equal(check_edit(base), full["logits"])
    for names in (["mask"], ["bias", "bias_token"], ["bias", "bias_token", "nbias"], ["text", "len", "repetition"],
                  ["text", "len", "prompt", "frequency"], ["text", "len", "presence"], ["token", "presence"],
                  ["token", "parent", "frequency", "repetition"], ["nodes"], ["text", "len", "token", "nodes", "parent", "presence"]):
        check_edit({**base, **{n: full[n] for n in names}})


def test_edit_many_rows_of_one_text():
    """More rows than a tree has nodes, without their tokens."""
    c = edit_case(6, 2, 200, 300, 30, token=False)
    check_edit(c)


def test_edit_special_values():
    c = edit_case(7, 2, 2, 500, 60, 5, True, few=30)
    c["logits"][:, 3], c["logits"][:, 4], c["logits"][:, 5] = np.inf, -np.inf, np.nan
    c["mask"][:] = 0xFFFFFFFF
    c["mask"][1, 0] = 0xFFFFFFF0
    c["text"][:, :9] = [3, 4, 5, -1, 500, 2 ** 31 - 1, -2 ** 31, 3, 7]
    c["token"][:, 0] = -1
    c["bias_token"][:, 0] = 10 ** 9
    c["len"][:], c["nodes"][:] = 60, 2
    got = ec.logits_edit_dev(**c)
    ok = np.isfinite(c["logits"])
    c["logits"][~ok] = 1.0
    with np.errstate(invalid="ignore"):
        want = check_edit(c)
    assert np.array_equal(got[:, 6:], want[:, 6:])
    assert np.isneginf(got[1, 3]) and np.isposinf(got[0, 3]) and np.isneginf(got[:, 4][[0, 2, 3]]).all()
    assert np.isnan(got[0, 5]) and np.isnan(got[3, 5])


@pytest.mark.parametrize("name,at,value", [("len", 1, -1), ("len", 1, 61), ("len", 1, 2 ** 31 - 1), ("nbias", 1, -1), ("nbias", 1, 6),
                                           ("nodes", 1, -1), ("nodes", 1, 9), ("parent", (1, 2), 2), ("parent", (1, 0), 0),
                                           ("parent", (1, 1), -2)])
def test_edit_bad_numbers(name, at, value):
    c = edit_case(8, 3, 8, 400, 60, 5)
    c["nodes"][1] = 6
    c[name][at] = value
    check_edit(c, bad=(1,))


def test_edit_in_place_and_strides():
    c = edit_case(9, 2, 3, 1001, 60, 5, True)
    want = check_edit(c)
    B, N, V, ld = 2, 3, 1001, 1024
    for odd in (0, 3):
        with ec._Call() as k:
            x = np.full((B * N + 1, ld), 3.5, np.float32)
            x.ravel()[odd:odd + B * N * ld].reshape(B * N, ld)[:, :V] = c["logits"]
            p = {n: k.put(n, c[n], t) for n, t in (
                ("text", np.int32), ("len", np.int32), ("prompt", np.int32), ("token", np.int32), ("nodes", np.int32),
                ("parent", np.int32), ("repetition", np.float32), ("frequency", np.float32), ("presence", np.float32),
                ("bias_token", np.int32), ("bias", np.float32), ("nbias", np.int32), ("mask", np.uint32))}
            a = k.put("x", x, np.float32) + 4 * odd
            rc = ec.lib().ec_logits_edit_dev(a, ld, a, ld, V, p["text"], 60, p["len"], p["prompt"], p["token"], p["nodes"], p["parent"],
                                             B, N, p["repetition"], p["frequency"], p["presence"], p["bias_token"], p["bias"],
                                             p["nbias"], 5, p["mask"], c["mask"].shape[1])
            assert rc == 0 and ec.lib().ec_sync() == 0
            got = k.get("x", np.float32, x.size)
        rows = got[odd:odd + B * N * ld].reshape(B * N, ld)
        assert (rows[:, V:] == 3.5).all() and (got[:odd] == 3.5).all()
        live = np.concatenate([np.arange(N) < n for n in c["nodes"]])
        assert np.array_equal(rows[live, :V], want[live]) and np.array_equal(rows[~live, :V], c["logits"][~live])


# ---------------------------------------------------------------------------
# together
# ---------------------------------------------------------------------------

class _Serve:
    """One layer's serving steps on device buffers: rows into the pages, attention, a
    language-model head, edited logits, sampling; and the texts read back."""
    H, KVH, hd, V, B, page, per = 6, 2, 64, 501, 5, 16, 20

    def __init__(self, seed, type, M, rows):
        s, r = self, np.random.default_rng(seed)
        s.rng, s.type, s.M, s.rows, s.T = r, type, M, rows, 40
        E = s.H * s.hd
        s.k = k = ec._Call()
        s.head = r.normal(0, 0.06, (s.V, E)).astype(np.float16)
        s.kg = r.normal(1, 0.2, s.hd).astype(np.float32)
        s.inv = ec.rope_inv_freq(s.hd, 1e4)
        s.pages = random_pages(r, type, s.KVH, s.hd, s.page, [s.per * s.page] * s.B)
        s.cache = s.pages.put(k)
        for n, a, t in (("head", s.head.view(np.uint16), np.uint16), ("kg", s.kg, np.float32), ("inv", s.inv, np.float64),
                        ("x", np.zeros((M, (s.H + 2 * s.KVH) * s.hd)), np.float32), ("q", np.zeros((M, E)), np.float32),
                        ("att", np.zeros((M, E)), np.float32), ("logits", np.zeros((M, s.V)), np.float32),
                        ("edited", np.zeros((M, s.V)), np.float32), ("token", np.zeros(M), np.int32),
                        ("start", np.zeros(s.B + 1), np.int32), ("past", np.zeros(s.B), np.int32), ("zero", np.zeros(s.B), np.int32),
                        ("total", np.zeros(s.B), np.int32), ("text", np.zeros((M, s.T)), np.int32), ("len", np.zeros(M), np.int32),
                        ("rep", np.full(M, 1.2), np.float32), ("freq", np.full(M, 0.3), np.float32),
                        ("u", np.zeros(M), np.float64), ("kc", np.zeros((s.B, s.per * s.page, s.KVH * s.hd)), np.uint16),
                        ("vc", np.zeros((s.B, s.per * s.page, s.KVH * s.hd)), np.uint16)):
            k.put(n, a, t)

    def new(self):
        s, r, M = self, self.rng, self.M
        n = np.ones(s.B, int) if s.rows == 1 else r.multinomial(r.integers(M // 2, M + 1), np.ones(s.B) / s.B)
        s.n, s.start = n, np.concatenate(([0], np.cumsum(n))).astype(np.int32)
        s.past = r.integers(0, s.per * s.page - n.max() + 1, s.B).astype(np.int32)
        s.total = (s.past + n).astype(np.int32)
        s.x = r.normal(0, 2, (M, (s.H + 2 * s.KVH) * s.hd)).astype(np.float32)
        s.text, s.len, s.u = r.integers(0, 60, (M, s.T)).astype(np.int32), r.integers(0, s.T + 1, M).astype(np.int32), r.random(M)
        for m in ("x", "start", "past", "total", "text", "len", "u"):
            a = np.ascontiguousarray(getattr(s, m))
            assert ec.lib().ec_memcpy_h2d(s.k.ptr(m), a.ctypes.data, a.nbytes) == 0

    def call(self):
        s, L, p, M = self, ec.lib(), self.k.ptr, self.M
        E, W, V, cache = s.H * s.hd, (s.H + 2 * s.KVH) * s.hd, s.V, C.byref(s.cache)
        return (L.ec_paged_append_dev(cache, p("x"), W, p("q"), E, s.H, None, p("kg"), 1e-6, p("inv"), s.hd, 0, 1.0, p("start"),
                                      p("past"), s.B, M)
                or L.ec_attention_paged_dev(cache, p("q"), E, s.H, p("start"), p("past"), s.B, M, s.per * s.page, 100, 4, p("att"), E)
                or L.ec_gemm_fp16_fp32_dev(p("logits"), p("att"), p("head"), M, E, V)
                or L.ec_logits_edit_dev(p("logits"), V, p("edited"), V, V, p("text"), s.T, p("len"), None, None, None, None, M, 1,
                                        p("rep"), p("freq"), None, None, None, None, 0, None, 0)
                or L.ec_sample_dev(p("edited"), M, V, V, None, None, None, None, p("u"), p("token"), None)
                or L.ec_paged_read_dev(cache, p("zero"), p("total"), s.B, s.per * s.page, p("kc"), p("vc"), s.B, s.per * s.page, None,
                                       None))

    def outputs(self):
        s, g, live = self, self.k.get, self.start[-1]
        pages = s.pages.got(s.k)
        return [g("q", np.uint32, (s.M, s.H * s.hd))[:live], g("att", np.uint32, (s.M, s.H * s.hd))[:live],
                g("edited", np.uint32, (s.M, s.V))[:live], g("token", np.int32, s.M)[:live], pages.k, pages.v,
                g("kc", np.uint16, s.B * s.per * s.page * s.KVH * s.hd), g("vc", np.uint16, s.B * s.per * s.page * s.KVH * s.hd)]


@pytest.mark.parametrize("type", TYPES)
@pytest.mark.parametrize("M,rows", [(5, 1), (90, 0)])
def test_serve_together(type, M, rows):
    """The operators in a row against the plain ones in a row, each on the device's own
    input to it."""
    s = _Serve(1, type, M, rows)
    try:
        for _ in range(3):
            s.new()
            before = s.pages.got(s.k)
            assert s.call() == 0, ec.last_error()
            assert ec.lib().ec_sync() == 0
            H, KVH, hd, live = s.H, s.KVH, s.hd, s.start[-1]
            q, after = check_append(dict(H=H, past=s.past, new=s.n, start=s.start, pages=before, qkv=s.x, qg=None, kg=s.kg), s.inv)
            now = s.pages.got(s.k)
            for n in ("k", "v") + (() if type == "fp16" else ("k_scale", "v_scale")):
                assert np.array_equal(getattr(now, n), getattr(after, n))
            assert np.array_equal(s.k.get("q", np.float32, (M, H * hd))[:live], q[:live])
            att = s.k.get("att", np.float32, (M, H * hd))
            one = np.concatenate((att[:live], np.full((1, H * hd), 7.25, np.float32)))
            check(dict(H=H, past=s.past, new=s.n, start=s.start, pages=now, q=q), 100, 4, got=one)
            logits = s.k.get("logits", np.float32, (M, s.V))
            assert np.abs(logits[:live] - att[:live].astype(np.float64) @ s.head.T.astype(np.float64)).max() < 1e-4
            edited = s.k.get("edited", np.float32, (M, s.V))
            check_edit(dict(logits=logits[:live], N=1, text=s.text[:live], len=s.len[:live],
                            repetition=np.full(live, 1.2, np.float32), frequency=np.full(live, 0.3, np.float32)), got=edited[:live])
            token = s.k.get("token", np.int32, M)
            for m in range(live):
                assert token[m] == ref_sample(edited[m], s.u[m])[0]
            for n in ("k", "v"):
                got = half(s.k.get(n + "c", np.uint16, (s.B, s.per * s.page, KVH, hd)))
                for b in range(s.B):
                    assert np.array_equal(got[b, :s.total[b]], rows_of(now, n, b, s.total[b]))
    finally:
        s.k.__exit__()


def test_serve_captured():
    """Graphs of single tokens and of chunks (they share the library's workspace),
    replayed in turn with new inputs, eager calls and larger ones between: the eager results."""
    L = ec.lib()
    a, b = _Serve(2, "int8", 5, 1), _Serve(3, "fp16", 90, 0)
    big = attn_case(50, "e4m3", 12, 2, 128, 16, [6000, 10, 3000], [40, 200, 1])
    graphs = []
    try:
        for s in (a, b):
            s.new()
            assert s.call() == 0 and L.ec_sync() == 0
        graphs = [_Graph(a.call), _Graph(b.call)]
        for turn in range(4):
            want = []
            for s in (a, b):
                s.new()
                assert s.call() == 0 and L.ec_sync() == 0  # a second pass over the same pages writes the same
                want.append(s.outputs())
            graphs[turn % 2].replay()
            graphs[1 - turn % 2].replay()
            assert L.ec_sync() == 0
            for s, w in zip((a, b), want):
                for x, y in zip(s.outputs(), w):
                    assert np.array_equal(x, y)
            check(big, rows=[(0, 3), (1, 150), (2, 0)])
    finally:
        for g in graphs:
            g.close()
        a.k.__exit__()
        b.k.__exit__()


def test_paged_text_into_drafted_tokens():
    """A text that was written in 8 bits, read into a slot, goes on with the operators for
    drafted tokens: its last token's attention is the same by both."""
    H, KVH, hd, n = 6, 2, 64, 300
    c = append_case(60, "int8", H, KVH, hd, 16, [0], [n], pad=0)
    q, pages = check_append(c, ec.rope_inv_freq(hd, 1e4))
    paged = ec.attention_paged_dev(pages, q, H, [0], [0, n])
    z = np.zeros((2, n, KVH * hd), np.uint16)
    kc, vc = ec.paged_read_dev(pages, z, z, [0], [n], [1])
    slot = ec.attention_tree_dev(q[-1:], kc, vc, H, KVH, [n - 1], 1, [1])
    # both are within 1e-6 of the same sums
    assert np.abs(slot - paged[-1:]).max() < 4e-6


def test_profiled_calls():
    import json
    s = _Serve(4, "e4m3", 90, 0)
    L = ec.lib()
    try:
        s.new()
        assert L.ec_prof_start(b"") == 0 and s.call() == 0
        buf = C.create_string_buffer(1 << 16)
        assert L.ec_prof_stop(buf, len(buf)) > 0
        names = {r["kernel"] for r in json.loads(buf.value.decode())}
        assert {"paged_append", "attention_paged", "logits_edit", "paged_read"} <= names
    finally:
        s.k.__exit__()
