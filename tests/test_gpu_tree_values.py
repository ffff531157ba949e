"""Tree attention over values like a model's: a token that takes most of a row's
weight, in front of a long text of small weights and of values with a mean; scores
that pass the maximum so far by tens; queries of every size.

Each row is compared with 64 bits, and the error with that of the same formula in
plain fp32 (numpy) on the same inputs."""
import math

import numpy as np
import pytest

import edgecore_amd as ec
from test_gpu_tree_ops import f16, lineage, trees

pytestmark = pytest.mark.gpu


def peaked(seed, H, KVH, hd, B, N, past, at, gap, slots=None, mixed=False, size=1.0, value=0.02):
    """Keys of which one, at place `at` (a share of the text, or "node": the first
    node), points where the queries do: its score stands about gap above the sum of
    the others' weights.  mixed: away from the queries of every second head.  size:
    of the queries; the keys are as much smaller."""
    rng = np.random.default_rng(seed)
    nslots, n = slots or B, past + N
    d = rng.choice([-1.0, 1.0], (KVH, hd))
    q = rng.normal(0, 1, (B * N, H, hd)) + np.repeat(d, H // KVH, 0)
    if mixed:
        q[:, 1::2] -= 2 * np.repeat(d, H // KVH, 0)[1::2]
    k = rng.standard_normal((nslots, n, KVH, hd), np.float32)
    v = rng.standard_normal((nslots, n, KVH, hd), np.float32) + np.float32(0.5)
    row = past if at == "node" else min(int(at * past), past - 1)
    # the others' weights sum to n e^(variance / 2), scores of variance |q|^2 / hd = 2
    k[:, row] = d * (math.log(n) + 1.0 + gap) / math.sqrt(hd)
    v[:, row] = rng.normal(0, value, (nslots, KVH, hd))
    return dict(H=H, KVH=KVH, N=N, past=np.full(B, past, np.int32), q=(q * size).reshape(B * N, H * hd).astype(np.float32),
                kc=f16(k / size).reshape(nslots, n, KVH * hd), vc=f16(v).reshape(nslots, n, KVH * hd),
                slot=(np.arange(B) % nslots).astype(np.int32), parent=trees(rng, B, N))


def attend(x, v, dt):
    x = x.astype(dt)
    w = np.exp(x - x.max(-1, keepdims=True))
    return (w @ v.astype(dt)) / w.sum(-1, keepdims=True, dtype=dt)


def check(c, rows, window=0):
    """Root mean squares of the errors over all the rows' elements: at most four times
    plain fp32's and 2^-20 of the outputs'.  (The score of a position that takes a
    share s of the weight is some 20 in units of log2, and half a step of it 2^-20:
    each of its sums, 4 to 8, is off by that, independently, in all by 2^-18 for
    the largest heads; it moves the output by s (1 - s) <= 1/4 of what lies between
    the values.  Small weights are off by 2^-36 of the largest at most, either way:
    32600 of them come to 2^-28 together.)"""
    H, KVH, N = c["H"], c["KVH"], c["N"]
    hd, G = c["q"].shape[1] // H, H // KVH
    got = ec.attention_tree_dev(c["q"], c["kc"], c["vc"], H, KVH, c["past"], N, c["slot"], None, c["parent"], window)
    err = plain = size = 0.0
    for b, i in rows:
        past = int(c["past"][b])
        line = lineage(list(c["parent"][b]))[i]
        lo = max(0, past + len(line) - window) if window else 0
        at = list(range(min(lo, past), past)) + [past + j for j in (line[-window:] if window else line)]
        for h in range(KVH):
            k, v = (c[m][c["slot"][b], at, h * hd:(h + 1) * hd].view(np.float16) for m in ("kc", "vc"))
            heads = slice(h * G * hd, (h + 1) * G * hd)
            q = c["q"][b * N + i, heads].reshape(G, hd)
            want = attend(q.astype(np.float64) @ k.astype(np.float64).T / math.sqrt(hd), v, np.float64)
            f32 = attend(q @ k.astype(np.float32).T * np.float32(1 / math.sqrt(hd)), v, np.float32)
            err += ((got[b * N + i, heads].reshape(G, hd) - want) ** 2).sum()
            plain += ((f32 - want) ** 2).sum()
            size += (want ** 2).sum()
    err, plain, size = (math.sqrt(x) for x in (err, plain, size))
    print("error %.2e, plain fp32 %.2e of the outputs" % (err / size, plain / size))
    assert err <= 4 * plain + 2.0 ** -20 * size, (err / size, plain / size)


SHAPES = [(14, 2, 64), (12, 2, 128), (16, 4, 96), (8, 1, 32), (5, 1, 40)]


@pytest.mark.parametrize("H,KVH,hd", SHAPES)
@pytest.mark.parametrize("N,past", [(1, 1000), (16, 4000), (64, 1000)])
@pytest.mark.parametrize("gap", [0.0, 2.0, 4.6])
def test_first_token_takes_most(H, KVH, hd, N, past, gap):
    """Shares of about 1/2, 0.9 and 0.99, the text in several parts."""
    check(peaked(int(10 * gap) + N, H, KVH, hd, 2, N, past, 0.0, gap), [(0, 0), (1, N - 1)])


@pytest.mark.parametrize("H,KVH,hd,N", [(14, 2, 64, 64), (12, 2, 128, 1)])
@pytest.mark.parametrize("gap", [0.0, 2.0, 4.6])
def test_first_token_of_a_long_text(H, KVH, hd, N, gap):
    check(peaked(int(10 * gap) + N, H, KVH, hd, 2, N, 32600, 0.0, gap), [(0, 0), (1, N - 1)])


@pytest.mark.parametrize("H,KVH,hd,past", [(12, 12, 64, 1000), (12, 12, 64, 2000), (12, 12, 64, 32600), (32, 8, 128, 2000),
                                           (32, 8, 128, 32600), (24, 12, 96, 2000), (48, 24, 32, 2000)])
@pytest.mark.parametrize("gap", [0.0, 2.0, 4.6])
def test_first_token_of_unsplit_texts(H, KVH, hd, past, gap):
    """Batches that fill the chip with one block per sequence and KV head."""
    check(peaked(past + int(10 * gap), H, KVH, hd, 70, 1, past, 0.0, gap, slots=2), [(0, 0), (69, 0)])


@pytest.mark.parametrize("H,KVH,hd,B", [(14, 2, 64, 2), (12, 2, 128, 2), (12, 12, 64, 70), (5, 1, 40, 2)])
@pytest.mark.parametrize("at", [0.0, 0.5, 0.97, 1.0, "node"])
@pytest.mark.parametrize("gap", [-3.0, 5.0, 20.0])
@pytest.mark.parametrize("mixed", [False, True])
def test_maximum_that_moves(H, KVH, hd, B, at, gap, mixed):
    """The position with the largest score in the first tile, the middle, the last
    tiles of the text or among the nodes, up to 30 above what came before; of all
    rows of a wave, or of every second one (where it weighs nothing for the others)."""
    N = 1 if B > 2 else 9
    check(peaked(B + N, H, KVH, hd, B, N, 1500, at, gap, slots=2, mixed=mixed, value=1.0), [(0, 0), (B - 1, N - 1)])


@pytest.mark.parametrize("H,KVH,hd", [(14, 2, 64), (12, 2, 128), (8, 1, 32)])
@pytest.mark.parametrize("size", [2.0 ** -12, 2.0 ** -9, 64.0, 2.0 ** 13])
def test_sizes_of_queries(H, KVH, hd, size):
    """Queries below 2^-4 and above 2^15 in units of the exponent (the latter against keys
    of 2^-13, whose 11 bits end at 2^-24), the keys as much larger or smaller."""
    for at, mixed in ((0.0, False), (0.6, True)):
        check(peaked(7, H, KVH, hd, 2, 9, 700, at, 3.0, mixed=mixed, size=size), [(0, 0), (1, 8)])


@pytest.mark.parametrize("H,KVH,hd", [(14, 2, 64), (12, 2, 128)])
def test_rows_of_unlike_sizes(H, KVH, hd):
    """Rows of one wave from 2^-40 to 2^17."""
    c = peaked(9, H, KVH, hd, 2, 9, 900, 0.4, 3.0)
    c["q"] = (c["q"].reshape(18, H, hd) * 2.0 ** np.resize([0, -40, 17, 0, -9, 2, 5], 18 * H).reshape(18, H, 1)
              ).reshape(18, H * hd).astype(np.float32)
    check(c, [(0, i) for i in range(9)] + [(1, 4)])


@pytest.mark.parametrize("window", [500, 1200])
def test_first_token_in_and_out_of_a_window(window):
    """The row that takes the weight in front of the window, and at its edge."""
    for H, KVH, hd in ((14, 2, 64), (12, 2, 128)):
        for at in (0.0, 1.0 - window / 3000, 1.0 - (window - 4) / 3000):
            check(peaked(window, H, KVH, hd, 2, 9, 3000, at, 4.6), [(0, 0), (1, 8)], window)


@pytest.mark.parametrize("H,KVH,hd", [(14, 2, 64), (12, 2, 128), (8, 1, 32), (5, 1, 40)])
@pytest.mark.parametrize("at", [100, 703])
def test_infinite_keys_and_queries(H, KVH, hd, at):
    """One element of a key that is seen (in the text, among the nodes) is infinite: NaN
    where the score is +inf; where it is -inf, NaN or the result without the key.  One
    of a query: NaN in its own row and head."""
    c = peaked(11, H, KVH, hd, 2, 5, 703, 0.3, 1.0)
    c["parent"][:] = np.arange(5) - 1
    call = lambda: ec.attention_tree_dev(c["q"], c["kc"], c["vc"], H, KVH, c["past"], 5, c["slot"], None, c["parent"])
    clean = call().reshape(2, 5, KVH, H // KVH, hd)
    e = hd // 2 + 3
    kept = c["kc"][0, at].copy()
    for sign in (1, -1):
        c["kc"][0, at] = kept
        c["kc"][0, at, e] = 0x7C00 if sign > 0 else 0xFC00
        got = call().reshape(clean.shape)
        up = c["q"].reshape(clean.shape)[0, :, 0, :, e] * sign > 0
        assert up.any() and not up.all()
        assert np.isnan(got[0, :, 0][up]).all()
        # the same with a key whose score is far below all others
        far = c["q"].reshape(clean.shape)[0, :, 0][~up]
        for n, q in zip(np.argwhere(~up), far):
            i, g = n
            mine = got[0, i, 0, g]
            if np.isnan(mine).all():
                continue
            keys, values = (c[m][0, :703 + i + 1, :hd].view(np.float16).astype(np.float64) for m in ("kc", "vc"))
            with np.errstate(invalid="ignore"):
                x = keys @ q.astype(np.float64) / math.sqrt(hd)
            x[at] = -np.inf
            # (7e2 positions, values of about 1: what plain fp32 is off by stays below 1e-5)
            assert np.abs(mine - attend(x[None], values, np.float64)[0]).max() < 1e-5
        assert np.array_equal(got[1], clean[1]) and np.array_equal(got[0, :, 1:], clean[0, :, 1:])
    c["kc"][0, at] = kept
    for bad in (np.inf, -np.inf, np.nan):
        q = c["q"][3, hd + 1]
        c["q"][3, hd + 1] = bad
        got = call().reshape(10, H, hd)
        c["q"][3, hd + 1] = q
        assert np.isnan(got[3, 1]).all()
        got[3, 1] = clean.reshape(10, H, hd)[3, 1]
        # (when a row's maximum moves decides when its neighbours' do, by their room)
        assert np.abs(got - clean.reshape(10, H, hd)).max() < 1e-5
