"""The operators for drafted tokens (sampling, normed and rotated appends, tree
attention, accepted rows) against plain 64-bit implementations, at the sizes,
masks and values where they can go wrong.

Tolerances are worst-case bounds of the 32-bit arithmetic, written where they
are used; whole numbers and copied rows are equal."""
import ctypes as C
import math

import numpy as np
import pytest

import edgecore_amd as ec

pytestmark = pytest.mark.gpu

U = 2.0 ** -24  # half a step of fp32
NAN16, INF16 = 0x7E00, 0x7C00


def f16(x):
    return np.asarray(x, np.float32).astype(np.float16).view(np.uint16)


def trees(rng, B, N, reach=4):
    at = np.arange(N)
    return np.where(at == 0, -1, np.maximum(at - rng.integers(1, reach + 1, (B, N)), 0)).astype(np.int32)


def lineage(parent):
    up = []
    for i, p in enumerate(parent):
        up.append((up[p] if p >= 0 else []) + [i])
    return up


def lines_of(parent, b, N):
    return lineage(range(-1, N - 1) if parent is None else list(parent[b][:N]))


# ---------------------------------------------------------------------------
# sampling
# ---------------------------------------------------------------------------

def ref_sample(x, u, T=1.0, k=0, p=1.0, q=0.0):
    """One row's (token, probability) from the definition, in 64 bits."""
    x = np.where(np.isnan(x), -np.inf, x.astype(np.float64)) + 0.0
    top = x.max()
    if top == -np.inf:
        return -1, 0.0
    if not T > 0:
        return int(np.argmax(x)), 1.0
    with np.errstate(invalid="ignore", over="ignore", under="ignore", divide="ignore"):
        w = np.where(x == top, 1.0, np.where((x == -np.inf) | (top == np.inf), 0.0, np.exp((x - top) / T)))
    order = np.argsort(-x, kind="stable")
    if 0 < k:
        order = order[:k]
    order = order[w[order] > 2.0 ** -45]  # what is left out weighs 2^-27 of the largest in all, at most
    c = np.cumsum(w[order])
    if p < 1.0:
        order = order[:max(1, int((c - w[order] < p * c[-1]).sum()))]
    if q > 0.0:
        order = order[:max(1, int((w[order] >= min(q, 1.0)).sum()))]
    c = np.cumsum(w[order])
    j = min(int((c <= u * c[-1]).sum()), len(order) - 1)
    return int(order[j]), w[order[j]] / c[-1]


def check_sample(x, u, T=None, k=None, p=None, q=None, vocab=None):
    R = len(x)
    tok, prob = ec.sample_dev(x, u, T, k, p, q, vocab)
    for r in range(R):
        want = ref_sample(x[r, :vocab], u[r], *(d if a is None else type(d)(a[r]) for a, d in
                                                 ((T, 1.0), (k, 0), (p, 1.0), (q, 0.0))))
        assert tok[r] == want[0], (r, tok[r], want)
        # one rounding to fp32, weights in steps of 2^-44
        assert abs(prob[r] - want[1]) <= 2 * U * want[1] + 1e-12, (r, prob[r], want)
    return tok, prob


def settings(rng, R):
    pick = rng.integers(0, 6, R)
    T = np.where(pick == 0, 0.0, rng.uniform(0.3, 2.0, R)).astype(np.float32)
    k = np.where(pick % 2 == 1, rng.integers(1, 300, R), 0).astype(np.int32)
    p = np.where(pick >= 3, rng.uniform(0.05, 1.0, R), 1.0).astype(np.float32)
    q = np.where(pick >= 4, rng.uniform(0.0001, 0.3, R), 0.0).astype(np.float32)
    return T, k, p, q


@pytest.mark.parametrize("V", [1, 2, 3, 63, 64, 65, 255, 1000, 1024, 1025, 4095, 4096, 4097, 5000, 50257, 151936])
def test_sample_sizes(V):
    rng = np.random.default_rng(V)
    R = 24 if V < 10000 else 12
    x = rng.normal(0, 2.5, (R, V)).astype(np.float32)
    check_sample(x, rng.random(R))
    check_sample(x, rng.random(R), *settings(rng, R))


@pytest.mark.parametrize("V", [40, 3000, 30011])
def test_sample_ties(V):
    """Logits of few values: the order among equal ones is by index, and borders
    fall inside them."""
    rng = np.random.default_rng(V + 1)
    R = 24
    x = (rng.integers(-3, 4, (R, V)) * 0.5).astype(np.float32)
    x[3] = 0.0
    x[4] = np.where(rng.random(V) < 0.5, 0.0, -0.0)
    x[5, V // 2:] = x[5].max()
    x[6] = 1e30
    T, k, p, q = settings(rng, R)
    k[3:7] = [V // 3, V // 2, 7, 0]
    check_sample(x, rng.random(R), T, k, p, q)
    check_sample(x, rng.random(R), None, None, p, None)


@pytest.mark.parametrize("V,step", [(60000, 2.0 ** -9), (60000, 2.0 ** -12), (151936, 2.0 ** -13), (151936, 2.0 ** -7)])
def test_sample_ties_in_full_bins(V, step):
    """Logits on a grid: bins of hundreds of elements, equal ones by a few to hundreds."""
    rng = np.random.default_rng(int(V + 1 / step))
    R = 12
    x = (np.round(rng.normal(0, 1.5, (R, V)) / step) * step).astype(np.float32)
    T = rng.uniform(0.8, 3.0, R).astype(np.float32)
    check_sample(x, rng.random(R), T)
    check_sample(x, rng.random(R), T, None, rng.uniform(0.3, 0.99, R).astype(np.float32))
    check_sample(x, rng.random(R), T, rng.integers(V // 50, V // 2, R).astype(np.int32), None,
                 np.where(rng.random(R) < 0.5, 1e-3, 0.0).astype(np.float32))


def test_sample_special_values():
    rng = np.random.default_rng(3)
    V = 5003
    x = rng.normal(0, 2, (12, V)).astype(np.float32)
    x[0] = -np.inf                       # nothing left
    x[1] = np.nan
    x[2, 1:] = -np.inf                   # one token
    x[3, ::2] = -np.inf
    x[4, ::3] = np.nan
    x[5, [17, 4000]] = np.inf            # the infinite ones alone, equal
    x[6] = -np.inf
    x[6, 4999] = -3.0e38
    x[7] = np.finfo(np.float32).min      # masked by the lowest value everywhere
    x[8] = np.finfo(np.float32).min
    x[8, [5, 50]] = [1.0, 2.0]
    x[9] = np.finfo(np.float32).max
    x[10, :] = np.where(rng.random(V) < 0.5, np.finfo(np.float32).min, x[10])
    x[11, :4000] = -np.inf
    for seed in range(6):
        u = np.random.default_rng(seed).random(12)
        tok, prob = check_sample(x, u)
        assert tok[0] == tok[1] == -1 and tok[2] == 0 and tok[5] in (17, 4000) and prob[5] == 0.5 and tok[6] == 4999
        check_sample(x, u, k=np.full(12, 60, np.int32), p=np.full(12, 0.7, np.float32))
        check_sample(x, u, T=np.full(12, 0.8, np.float32), q=np.full(12, 0.05, np.float32))
        check_sample(x, u, k=np.full(12, 4500, np.int32))
        check_sample(x, u, T=np.zeros(12, np.float32))


@pytest.mark.parametrize("V", [64, 4096, 4100, 12289])
def test_sample_few_left(V):
    """Masks of -inf (or NaN) that leave one lane's tokens, a few or whole chunks; low
    temperatures, at which most weights are 0."""
    rng = np.random.default_rng(V + 3)
    x = rng.normal(0, 2, (8, V)).astype(np.float32)
    at = np.arange(V)
    x[0, at % 64 != 5] = -np.inf
    x[1, at % 64 != 63] = np.nan
    x[2, at != V - 1] = -np.inf
    x[3, :V // 2] = -np.inf
    x[4, V // 2:] = np.nan
    x[5, rng.random(V) < 0.999] = -np.inf
    x[5, 3] = 0.0
    x[6] *= 40.0
    T = np.array([1, 1, 1, 0.7, 0.7, 1, 1, 0.01], np.float32)
    for u in (0.0, 0.3, 0.9999):
        check_sample(x, np.full(8, u), T)
        check_sample(x, np.full(8, u), T, np.full(8, 3, np.int32), np.full(8, 0.9, np.float32), np.full(8, 0.01, np.float32))


@pytest.mark.parametrize("V", [37, 6000])
def test_sample_extreme_settings(V):
    rng = np.random.default_rng(V + 2)
    vals = [dict(T=t) for t in (np.inf, 1e30, 1e-30, 1e-42, 1e-3, 50.0, -1.0, np.nan, -np.inf)]
    vals += [dict(k=k) for k in (-5, 0, 1, 2, V - 1, V, V + 1, 1 << 30)]
    vals += [dict(p=p) for p in (-1.0, 0.0, 1e-30, 1e-6, 0.5, 0.999999, 1.0, 2.0, np.nan)]
    vals += [dict(q=q) for q in (-1.0, 0.0, 1e-30, 1e-6, 0.5, 1.0, 3.0, np.nan)]
    R = len(vals)
    x = rng.normal(0, 2, (R, V)).astype(np.float32)
    x[:, 1] = x[:, 0]
    a = {n: np.array([v.get(n, d) for v in vals], t) for n, d, t in
         (("T", 1.0, np.float32), ("k", 0, np.int32), ("p", 1.0, np.float32), ("q", 0.0, np.float32))}
    for u in (0.0, 2.0 ** -60, 0.25, 0.999, 1.0 - 2.0 ** -53):
        check_sample(x, np.full(R, u), **a)
    # outside [0, 1) the first and the last of those that stay
    for u, want in ((-1.0, 0.0), (1.0, 1.0 - 2.0 ** -53), (7.0, 1.0 - 2.0 ** -53), (np.nan, 1.0 - 2.0 ** -53)):
        got = ec.sample_dev(x, np.full(R, u), a["T"], a["k"], a["p"], a["q"])
        assert np.array_equal(got[0], ec.sample_dev(x, np.full(R, want), a["T"], a["k"], a["p"], a["q"])[0])


def test_sample_stride_and_repeats():
    """Rows inside wider ones (odd addresses among them); the same call twice."""
    rng = np.random.default_rng(9)
    x = rng.normal(0, 2, (9, 2049)).astype(np.float32)
    x[:, 2001:] = 100.0
    u = rng.random(9)
    a, b = (check_sample(x, u, p=np.full(9, 0.9, np.float32), vocab=2001) for _ in range(2))
    assert np.array_equal(a[0], b[0]) and np.array_equal(a[1].view(np.uint32), b[1].view(np.uint32))


def test_sample_many_rows():
    """More rows than a batch takes."""
    rng = np.random.default_rng(17)
    V = 9000  # 3 chunks: 2730 rows a batch
    x = np.tile(rng.normal(0, 2, (60, V)).astype(np.float32), (50, 1))
    u = rng.random(len(x))
    T = rng.uniform(0.2, 1.5, len(x)).astype(np.float32)
    tok, prob = ec.sample_dev(x, u, T)
    for r in [*range(0, 60), *range(2700, 2760), *range(2990, 3000)]:
        want = ref_sample(x[r], u[r], T[r])
        assert tok[r] == want[0] and abs(prob[r] - want[1]) <= 2 * U * want[1] + 1e-12


def test_sample_unlikely_tokens():
    """Drawn tokens of small weights: their probability to 2^-45 of the largest weight;
    those that weigh less than half a step are never drawn."""
    V, at = 5000, 4321
    gaps = np.array([5.0, 10.0, 15.0, 20.0, 25.0, 28.0, 30.0, 30.4])
    x = np.full((len(gaps), V), -1000.0, np.float32)
    x[:, 17], x[:, at] = 3.0, 3.0 - gaps
    got = ec.sample_dev(x, np.full(len(gaps), 1.0 - 2.0 ** -53))
    w = np.exp((x[:, at].astype(np.float64) - 3.0))
    assert (got[0] == at).all()
    # half a step of the weight (and the exponential's own 2^-46 of it), one rounding to fp32
    assert (np.abs(got[1] / (w / (1 + w)) - 1) <= 2.0 ** -45 / w + 2.0 ** -46 + 2 * U).all()
    x[:, at] = 3.0 - 31.3
    assert (ec.sample_dev(x, np.full(len(gaps), 1.0 - 2.0 ** -53))[0] == 17).all()


def test_sample_as_the_driver():
    """With top_k alone and the driver's number the driver's token."""
    rng = np.random.default_rng(12)
    x = rng.normal(0, 3, (40, 50257)).astype(np.float32)
    state, u, want = 42, [], []
    for r in range(40):
        st = C.c_ulonglong(state)
        u.append(ec.lib().ec_rng_next(C.byref(st)) / 0xFFFFFFFF)
        tok, state = ec.sample_full(x[r], 0.8, 40, state)
        want.append(tok)
    got, _ = ec.sample_dev(x, np.array(u), np.full(40, 0.8, np.float32), np.full(40, 40, np.int32))
    assert list(got) == want


def test_sample_frequencies():
    """20000 numbers of a regular grid through one row: each token as often as
    its probability says, to the one number at either of its borders."""
    rng = np.random.default_rng(13)
    n, V = 20000, 50
    row = rng.normal(0, 1.5, V).astype(np.float32)
    got, _ = ec.sample_dev(np.tile(row, (n, 1)), (np.arange(n) + 0.5) / n)
    p = np.exp(row.astype(np.float64) - row.max())
    assert np.abs(np.bincount(got, minlength=V) - n * p / p.sum()).max() <= 1.0


# ---------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------

def attn_case(seed, H, KVH, hd, B, N, past, nslots=None, C=None, tree=True, nodes=None):
    rng = np.random.default_rng(seed)
    past = np.array(past, np.int32)
    nslots = nslots or B + 1
    C = C or int(past.max()) + N
    return dict(H=H, KVH=KVH, past=past, N=N, q=rng.normal(0, 1, (B * N, H * hd)).astype(np.float32),
                kc=f16(rng.normal(0, 1, (nslots, C, KVH * hd))), vc=f16(rng.normal(0, 1, (nslots, C, KVH * hd))),
                slot=rng.permutation(nslots)[:B].astype(np.int32), parent=trees(rng, B, N) if tree else None,
                nodes=None if nodes is None else np.array(nodes, np.int32))


def sees(c, b, i, window):
    """The cache rows that node i of sequence b sees."""
    line, past = lines_of(c["parent"], b, c["N"])[i], int(c["past"][b])
    lo = max(0, past + len(line) - window) if window else 0
    return list(range(min(lo, past), past)) + [past + j for j in (line[-window:] if window else line)]


def check_attention(c, window=0, rows=None, got=None, **k):
    H, KVH, N = c["H"], c["KVH"], c["N"]
    hd = c["q"].shape[1] // H
    out = np.full_like(c["q"], 7.25)
    if got is None:
        got = ec.attention_tree_dev(c["q"], c["kc"], c["vc"], H, KVH, c["past"], N, c["slot"], c["nodes"], c["parent"],
                                    window, out=out, **k)
    slots = np.arange(len(c["past"])) if c["slot"] is None else c["slot"]
    worst = se = sw = 0.0
    for b in range(len(c["past"])):
        n = N if c["nodes"] is None else c["nodes"][b]
        assert (got[b * N + n:(b + 1) * N] == 7.25).all()  # padding is as it was
        for i in range(n):
            if rows is not None and (b, i) not in rows:
                continue
            at = sees(c, b, i, window)
            kk = c["kc"][slots[b], at].view(np.float16).astype(np.float64).reshape(len(at), KVH, hd)
            vv = c["vc"][slots[b], at].view(np.float16).astype(np.float64).reshape(len(at), KVH, hd)
            q = c["q"][b * N + i].astype(np.float64).reshape(KVH, H // KVH, hd)
            x = np.einsum("kgd,nkd->kgn", q, kk) / math.sqrt(hd)
            size = np.einsum("kgd,nkd->kgn", np.abs(q), np.abs(kk)) / math.sqrt(hd)
            p = np.exp(x - x.max(-1, keepdims=True))
            p /= p.sum(-1, keepdims=True)
            want = np.einsum("kgn,nkd->kgd", p, vv)
            # a score is off by the roundings of its hd + 2 steps and of its q (2^-22 where
            # it is split in two 16-bit parts), a weight by twice that and its own
            # exponential's, the sum by one rounding a term
            dx = size * (hd + 8) * 2 * U + np.abs(x) * 4 * U
            tol = np.einsum("kgn,nkd->kgd", p * (2 * dx.max(-1, keepdims=True) + (len(at) + 16) * 2 * U), np.abs(vv)) + 1e-30
            err = np.abs(got[b * N + i].reshape(want.shape) - want)
            assert (err <= tol).all(), (b, i, err.max(), (err / tol).max())
            worst, se, sw = max(worst, (err / tol).max()), se + (err ** 2).sum(), sw + (want ** 2).sum()
            # independent roundings of hd + n terms (with 8 for chance): what a 16-bit
            # rounding of q or of the weights would pass 10 times over
    if sw:
        span = hd + int(c["past"].max()) + N
        assert math.sqrt(se / sw) <= 8 * U * math.sqrt(span), (math.sqrt(se / sw), worst)
    return got


HEADS = [(14, 2, 64), (12, 2, 128), (12, 12, 64), (16, 4, 96), (8, 1, 32), (3, 3, 20), (2, 1, 250), (5, 1, 7), (2, 2, 512),
         (6, 2, 256)]


@pytest.mark.parametrize("H,KVH,hd", HEADS)
@pytest.mark.parametrize("N,past", [(1, [0, 1, 63, 64, 65, 130]), (5, [0, 31, 200]), (16, [0, 500, 129]), (64, [190, 1])])
def test_attention_heads(H, KVH, hd, N, past):
    check_attention(attn_case(hd * N + H, H, KVH, hd, len(past), N, past))


@pytest.mark.parametrize("H,KVH,hd,N", [(14, 2, 64, 9), (12, 12, 64, 1), (12, 2, 128, 33), (3, 3, 20, 6)])
@pytest.mark.parametrize("window", [1, 2, 7, 64, 100, 333, 5000, 2147483647])
def test_attention_window(H, KVH, hd, N, window):
    check_attention(attn_case(window % 1000, H, KVH, hd, 4, N, [0, 3, 97, 700]), window)


@pytest.mark.parametrize("H,KVH,hd", [(14, 2, 64), (12, 2, 128), (12, 12, 64), (5, 1, 7)])
def test_attention_ragged_nodes_and_chains(H, KVH, hd):
    """Padding rows, sequences without nodes, chains, slot = sequence."""
    c = attn_case(5, H, KVH, hd, 5, 11, [20, 0, 77, 300, 64], nodes=[3, 0, 11, 1, 10])
    check_attention(c)
    c["parent"] = None
    check_attention(c)
    c["slot"] = None
    check_attention(c, window=9)
    c["nodes"] = None
    check_attention(c, max_past=300)


@pytest.mark.parametrize("H,KVH,hd,B,N,past,rows", [
    (14, 2, 64, 2, 64, [32600, 20011], [(0, 0), (0, 63), (1, 31), (1, 5)]),
    (12, 2, 128, 3, 16, [4000, 3001, 8190], [(0, 0), (1, 7), (2, 15)]),
    (12, 12, 64, 16, 1, [1000 - 7 * b for b in range(16)], None),
    (12, 2, 128, 1, 1, [16384], None),
    (2, 1, 250, 1, 3, [5000], None),
])
def test_attention_long(H, KVH, hd, B, N, past, rows):
    check_attention(attn_case(B + N, H, KVH, hd, B, N, past), rows=rows)


@pytest.mark.parametrize("H,KVH,hd", [(14, 2, 64), (12, 2, 128), (5, 1, 7)])
def test_attention_roots_and_wide_trees(H, KVH, hd):
    """Several roots, a star and a chain of 64."""
    c = attn_case(8, H, KVH, hd, 3, 64, [70, 0, 5])
    c["parent"][0] = -1
    c["parent"][1] = np.where(np.arange(64) == 0, -1, 0)
    c["parent"][2] = np.arange(64) - 1
    check_attention(c)
    check_attention(c, window=3)


@pytest.mark.parametrize("H,KVH,hd", [(14, 2, 64), (12, 2, 128), (12, 12, 64), (16, 4, 96), (5, 1, 7)])
def test_attention_unseen_values(H, KVH, hd):
    """NaN and infinities in rows that a node does not see (behind the nodes, in
    front of the window, other branches) do not reach it; in rows that it sees
    they do."""
    c = attn_case(21, H, KVH, hd, 2, 12, [150, 90], C=300, nodes=[12, 9])
    kc, vc = c["kc"], c["vc"]
    for b, n in ((0, 12), (1, 9)):
        s, p = c["slot"][b], c["past"][b]
        kc[s, p + n:], vc[s, p + n:] = NAN16, NAN16
    other = [s for s in range(3) if s not in c["slot"]][0]
    kc[other], vc[other] = INF16, NAN16
    clean = check_attention(c)
    # one node's row: those that do not see it keep their values
    j, s = 4, c["slot"][0]
    see = [j in line for line in lineage(list(c["parent"][0]))]
    for cache, bad in ((vc, NAN16), (vc, INF16), (kc, NAN16), (kc, INF16)):
        kept = cache[s, 150 + j].copy()
        cache[s, 150 + j] = bad
        got = ec.attention_tree_dev(c["q"], kc, vc, H, KVH, c["past"], 12, c["slot"], c["nodes"], c["parent"],
                                    out=np.full_like(c["q"], 7.25))
        cache[s, 150 + j] = kept
        for i in range(12):
            if see[i]:
                assert not np.isfinite(got[i]).all() or cache is kc
            else:
                assert np.allclose(got[i], clean[i], rtol=0, atol=1e-5), i
        assert np.array_equal(got[12:], clean[12:])
    # in front of the window of some nodes, not of others
    vc[c["slot"][0], 150 - 20 + 3], kc[c["slot"][1], :60] = INF16, NAN16
    c2 = dict(c)
    got = ec.attention_tree_dev(c["q"], kc, vc, H, KVH, c["past"], 12, c["slot"], c["nodes"], c["parent"], 20,
                                out=np.full_like(c["q"], 7.25))
    hit = [133 in sees(c2, 0, i, 20) for i in range(12)]
    assert any(hit) and not all(hit)
    for i in range(12):
        assert np.isfinite(got[i]).all() == (not hit[i]), i
    vc[c["slot"][0], 133] = f16(np.ones(KVH * hd))
    check_attention(c, window=20)


@pytest.mark.parametrize("H,KVH,hd", [(14, 2, 64), (12, 2, 128), (8, 1, 32), (5, 1, 7)])
def test_attention_seen_values(H, KVH, hd):
    """One element of a value that is not finite, in the text: the outputs of that
    element and its KV head are not finite, all others are as they were; of a key:
    the KV head's."""
    c = attn_case(22, H, KVH, hd, 2, 5, [700, 90])
    clean = check_attention(c)
    s, at, e = c["slot"][0], 300, (KVH - 1) * hd + hd // 2
    for cache, bad in ((c["vc"], NAN16), (c["vc"], INF16), (c["kc"], NAN16)):
        kept = cache[s, at, e]
        cache[s, at, e] = bad
        got = ec.attention_tree_dev(c["q"], c["kc"], c["vc"], H, KVH, c["past"], 5, c["slot"], None, c["parent"])
        cache[s, at, e] = kept
        hit = np.zeros((10, KVH, H // KVH, hd), bool)
        if cache is c["vc"]:
            hit[:5, -1, :, hd // 2] = True
        else:
            hit[:5, -1] = True
        hit = hit.reshape(10, H * hd)
        assert not np.isfinite(got[hit]).any() and np.array_equal(got[~hit], clean[~hit])


@pytest.mark.parametrize("H,KVH,hd,B,N", [(2, 1, 64, 130, 2), (4, 1, 128, 65, 3), (2, 1, 32, 200, 1), (6, 2, 64, 64, 1)])
@pytest.mark.parametrize("window", [0, 300])
def test_attention_many_ragged_sequences(H, KVH, hd, B, N, window):
    """More sequences than a wave has lanes, from empty to long ones, some of no
    nodes, one that takes no part: each has its share of the blocks."""
    rng = np.random.default_rng(B)
    past = rng.integers(0, 200, B)
    past[rng.integers(0, B, 5)] = [0, 3000, 1, 2047, 1500]
    nodes = rng.integers(0, N + 1, B)
    nodes[past > 1000] = N
    c = attn_case(B, H, KVH, hd, B, N, past, nodes=nodes)
    c["slot"][7], n7 = -1, int(c["nodes"][7])
    n = np.where(np.arange(B) == 7, 0, c["nodes"])
    got = ec.attention_tree_dev(c["q"], c["kc"], c["vc"], H, KVH, c["past"], N, c["slot"], c["nodes"], c["parent"], window,
                                out=np.full_like(c["q"], 7.25))
    assert np.isnan(got[7 * N:7 * N + n7]).all()
    got[7 * N:8 * N] = 7.25
    check_attention({**c, "nodes": n}, window, got=got)


@pytest.mark.parametrize("at,value", [((1, 0), 0), ((1, 3), 3), ((1, 7), -2), ((1, 7), 2 ** 31 - 1)])
@pytest.mark.parametrize("window", [0, 100])
def test_attention_bad_parents_in_a_long_text(at, value, window):
    """Splits whose tiles hold no node mark their rows too."""
    c = attn_case(32, 14, 2, 64, 3, 8, [2000, 3000, 700])
    want = check_attention(c, window, rows=[(0, 0), (2, 7)])
    c["parent"][at] = value
    got = ec.attention_tree_dev(c["q"], c["kc"], c["vc"], 14, 2, c["past"], 8, c["slot"], None, c["parent"], window)
    assert np.isnan(got[8:16]).all()
    assert np.array_equal(got[:8], want[:8]) and np.array_equal(got[16:], want[16:])


def test_attention_wide_scores():
    """Scores of thousands (one position takes all) and equal ones."""
    c = attn_case(4, 12, 2, 128, 2, 5, [300, 64])
    c["q"] *= 300.0
    got = ec.attention_tree_dev(c["q"], c["kc"], c["vc"], 12, 2, c["past"], 5, c["slot"], None, c["parent"])
    assert np.isfinite(got).all()
    c["q"][:] = 0.0
    check_attention(c)
    c["q"][:] = 1e-30
    check_attention(c)


BAD = [("slot", 1, 4), ("slot", 1, -1), ("slot", 1, 2 ** 31 - 1), ("past", 1, -1), ("past", 1, 95), ("past", 1, 2 ** 31 - 1),
       ("past", 1, -2 ** 31), ("nodes", 1, 9), ("nodes", 1, -1), ("nodes", 1, 2 ** 31 - 1), ("parent", (1, 0), 0),
       ("parent", (1, 3), 3), ("parent", (1, 3), 2 ** 31 - 1), ("parent", (1, 5), -2)]


@pytest.mark.parametrize("hd", [64, 20])
@pytest.mark.parametrize("name,at,value", BAD)
def test_attention_bad_numbers(hd, name, at, value):
    """A sequence whose numbers name no rows is NaN, the others are as they are."""
    c = attn_case(31, 4, 2, hd, 3, 8, [50, 60, 40], nslots=4, C=100, nodes=[8, 7, 8])
    want = check_attention(c)
    c[name][at] = value
    got = ec.attention_tree_dev(c["q"], c["kc"], c["vc"], 4, 2, c["past"], 8, c["slot"], c["nodes"], c["parent"],
                                out=np.full_like(c["q"], 7.25))
    n = 8 if name == "nodes" else 7
    assert np.isnan(got[8:8 + n]).all() and (got[8 + n:16] == 7.25).all()
    assert np.array_equal(got[:8], want[:8]) and np.array_equal(got[16:], want[16:])


def test_attention_max_past():
    c = attn_case(33, 4, 2, 64, 3, 4, [50, 60, 40])
    want = check_attention(c)
    got = ec.attention_tree_dev(c["q"], c["kc"], c["vc"], 4, 2, c["past"], 4, c["slot"], None, c["parent"], max_past=50)
    assert np.isnan(got[4:8]).all()
    assert np.allclose(got[:4], want[:4], rtol=0, atol=1e-5) and np.allclose(got[8:], want[8:], rtol=0, atol=1e-5)


@pytest.mark.parametrize("H,KVH,hd", [(14, 2, 64), (12, 2, 128)])
def test_attention_strides_and_alignment(H, KVH, hd):
    """Rows of q and out inside wider ones, and caches and rows at addresses that
    are multiples of 2 and 4 bytes alone."""
    c = attn_case(41, H, KVH, hd, 2, 6, [333, 64])
    E, M, L = H * hd, 12, ec.lib()
    nslots, Cr, kv = c["kc"].shape
    wide = np.full((M, E + 3), 9.0, np.float32)
    wide[:, :E] = c["q"]
    bufs = [ec.DeviceBuffer.from_array(np.concatenate([np.zeros(o, a.dtype), a.ravel()])) for a, o in
            ((wide, 1), (c["kc"], 1), (c["vc"], 3), (c["slot"], 0), (c["past"], 0), (c["parent"], 0),
             (np.full(M * (E + 5) + 8, 7.25, np.float32), 0))]
    try:
        for qo, ko, vo, oo in ((1, 1, 3, 1), (1, 1, 3, 0)):
            rc = L.ec_attention_tree_dev(bufs[0].ptr + 4 * qo, E + 3, bufs[1].ptr + 2 * ko, bufs[2].ptr + 2 * vo, nslots, Cr,
                                         H, KVH, hd, bufs[3].ptr, bufs[4].ptr, None, bufs[5].ptr, 2, 6, Cr, 0,
                                         bufs[6].ptr + 4 * oo, E + 5)
            assert rc == 0, ec.last_error()
            assert L.ec_sync() == 0
            raw = bufs[6].to_array(np.float32, M * (E + 5) + 8)
            o = raw[oo:oo + M * (E + 5)].reshape(M, E + 5)
            assert (o[:, E:] == 7.25).all()
            check_attention(c, got=np.ascontiguousarray(o[:, :E]))
            L.ec_memcpy_h2d(bufs[6].ptr, np.full_like(raw, 7.25).ctypes.data, raw.nbytes)
    finally:
        for b in bufs:
            b.close()


@pytest.mark.parametrize("H,KVH,hd,past", [(14, 2, 64, [900, 5]), (14, 2, 64, [9, 5]), (5, 1, 7, [90, 5])])
def test_attention_in_place(H, KVH, hd, past):
    """out = q, with splits and without."""
    c = attn_case(42, H, KVH, hd, 2, 6, past)
    want = check_attention(c)
    with ec._Call() as k:
        q, kc, vc = k.put("q", c["q"], np.float32), k.put("kc", c["kc"], np.uint16), k.put("vc", c["vc"], np.uint16)
        nslots, Cr, _ = c["kc"].shape
        E = H * hd
        rc = ec.lib().ec_attention_tree_dev(q, E, kc, vc, nslots, Cr, H, KVH, hd, *k.tree(c["slot"], c["past"], None, c["parent"]),
                                            2, 6, Cr, 0, q, E)
        assert rc == 0 and ec.lib().ec_sync() == 0
        assert np.array_equal(k.get("q", np.float32, (12, E)), want)


def test_attention_past_32_bits():
    """A slot whose rows lie more than 2^31 elements into the caches."""
    H, KVH, hd, Cr, N = 14, 2, 64, 32768, 3
    c = attn_case(43, H, KVH, hd, 1, N, [1500])
    kv, nslots = KVH * hd, 520
    L = ec.lib()
    row = 519 * Cr  # 519 * 32768 * 128 > 2^31
    assert row * kv > 2 ** 31
    kb, vb = ec.DeviceBuffer(2 * nslots * Cr * kv), ec.DeviceBuffer(2 * nslots * Cr * kv)
    small = [ec.DeviceBuffer.from_array(a) for a in (c["q"], np.array([519], np.int32), c["past"], c["parent"],
                                                      np.zeros_like(c["q"]))]
    try:
        for buf, a in ((kb, c["kc"]), (vb, c["vc"])):
            rows = np.ascontiguousarray(a[c["slot"][0]])
            assert L.ec_memcpy_h2d(buf.ptr + 2 * row * kv, rows.ctypes.data, rows.nbytes) == 0
        rc = L.ec_attention_tree_dev(small[0].ptr, H * hd, kb.ptr, vb.ptr, nslots, Cr, H, KVH, hd, small[1].ptr,
                                     small[2].ptr, None, small[3].ptr, 1, N, 2000, 0, small[4].ptr, H * hd)
        assert rc == 0 and L.ec_sync() == 0
        check_attention(c, got=small[4].to_array(np.float32, c["q"].shape))
    finally:
        for b in [kb, vb] + small:
            b.close()


# ---------------------------------------------------------------------------
# norm, rotation, append
# ---------------------------------------------------------------------------

def rope_case(seed, H, KVH, hd, B, N, past, nodes=None, tree=False, norm=True, C=None):
    rng = np.random.default_rng(seed)
    past = np.array(past, np.int32)
    C = C or int(past.max()) + N
    return dict(H=H, KVH=KVH, N=N, past=past, qkv=rng.normal(0, 3, (B * N, (H + 2 * KVH) * hd)).astype(np.float32),
                kc=f16(rng.normal(0, 1, (B + 1, C, KVH * hd))), vc=f16(rng.normal(0, 1, (B + 1, C, KVH * hd))),
                slot=rng.permutation(B + 1)[:B].astype(np.int32), parent=trees(rng, B, N) if tree else None,
                nodes=None if nodes is None else np.array(nodes, np.int32),
                qg=rng.normal(1, 0.3, hd).astype(np.float32) if norm else None,
                kg=rng.normal(1, 0.3, hd).astype(np.float32) if norm else None)


def check_rope(c, inv_freq=None, layout=0, factor=1.0, eps=1e-6, bad=()):
    H, KVH, N, B = c["H"], c["KVH"], c["N"], len(c["past"])
    hd = c["kc"].shape[2] // KVH
    M = B * N
    q0 = np.full((M, H * hd), 7.25, np.float32)
    got, kc, vc = ec.qk_norm_rope_dev(c["qkv"], c["kc"], c["vc"], H, KVH, c["past"], N, c["qg"], c["kg"], eps, inv_freq,
                                      layout, factor, c["slot"], c["nodes"], c["parent"], q0)
    rot = 0 if inv_freq is None else 2 * len(inv_freq)
    kw, vw = c["kc"].copy(), c["vc"].copy()
    x = c["qkv"].astype(np.float64).reshape(B, N, H + 2 * KVH, hd)
    tol_k = {}
    for b in range(B):
        n = N if c["nodes"] is None else c["nodes"][b]
        assert (got[b * N + n:(b + 1) * N] == 7.25).all()
        if b in bad:
            assert np.isnan(got[b * N:b * N + n]).all()
            continue
        lines = lines_of(c["parent"], b, N) if N <= 64 else None
        depth = np.array([len(lines[i]) - 1 if lines else i for i in range(n)], np.float64)
        ang = (c["past"][b] + depth)[:, None] * (inv_freq if rot else np.zeros(0))
        for first, heads, gamma in ((0, H, c["qg"]), (H, KVH, c["kg"])):
            y = x[b, :n, first:first + heads]
            if gamma is not None:
                y = y / np.sqrt((y ** 2).mean(-1, keepdims=True) + eps) * gamma
            z = y.copy()
            i0 = 2 * np.arange(rot // 2) if layout else np.arange(rot // 2)
            i1 = i0 + 1 if layout else i0 + rot // 2
            cs, sn = (factor * f(ang)[:, None, :] for f in (np.cos, np.sin))
            z[..., i0], z[..., i1] = y[..., i0] * cs - y[..., i1] * sn, y[..., i0] * sn + y[..., i1] * cs
            # the norm: hd roundings in the sum (half of it in the root) and four more;
            # the angle: reduced exactly, then one rounding of up to half a turn (pi
            # 2^-24), sine and cosine to two units; three roundings of the rotation
            size = np.abs(y)
            size[..., i0] = size[..., i1] = (np.abs(y[..., i0]) + np.abs(y[..., i1])) * abs(factor)
            tol = size * (hd / 2 + 14) * U + 1e-30
            if first == 0:
                err = np.abs(got[b * N:b * N + n].reshape(z.shape) - z)
                assert (err <= tol).all(), (b, err.max(), (err / tol).max())
            else:
                rows = slice(c["past"][b], c["past"][b] + n)
                g = kc[c["slot"][b], rows].view(np.float16).astype(np.float64).reshape(z.shape)
                err = np.abs(g - z)
                # one rounding to fp16 on top (2^-11, 2^-25 among the smallest)
                assert (err <= tol * 1.001 + np.abs(z) * 2.0 ** -11 + 2.0 ** -25).all(), (b, err.max())
                kw[c["slot"][b], rows] = kc[c["slot"][b], rows]
        rows = slice(c["past"][b], c["past"][b] + n)
        vw[c["slot"][b], rows] = f16(c["qkv"].reshape(B, N, H + 2 * KVH, hd)[b, :n, H + KVH:]).reshape(n, KVH * hd)
    assert np.array_equal(kc, kw) and np.array_equal(vc, vw)  # nothing else was written
    return got, kc, vc


@pytest.mark.parametrize("H,KVH,hd", [(14, 2, 64), (12, 2, 128), (12, 12, 64), (10, 5, 80), (16, 4, 96), (9, 3, 42), (3, 1, 256),
                                      (2, 2, 512), (2, 1, 7), (1, 1, 1)])
@pytest.mark.parametrize("layout", [0, 1])
def test_rope_heads(H, KVH, hd, layout):
    for N, past, norm in ((1, [0, 5, 70], True), (7, [3, 0, 40], False)):
        c = rope_case(hd + N, H, KVH, hd, 3, N, past, norm=norm)
        check_rope(c)
        for rot in {hd // 2 * 2, hd // 4 * 2, hd // 8 * 8, 2}:
            if 0 < rot <= hd:
                check_rope(c, ec.rope_inv_freq(rot, 1e4), layout)


@pytest.mark.parametrize("kind,factor", [(0, 1.0), (1, 1.1), (2, 1.0), (3, 1.0)])
def test_rope_far_positions(kind, factor):
    """Positions of a long context: the turns are formed in 64 bits."""
    inv = ec.rope_inv_freq(64, 1e4, kind, 8.0, 4096.0)
    check_rope(rope_case(3, 4, 2, 64, 3, 2, [32000, 131070, 60001]), inv, 0, factor)


@pytest.mark.parametrize("hd", [64, 128, 80, 42])
def test_rope_trees_and_padding(hd):
    c = rope_case(6, 6, 2, hd, 4, 33, [10, 0, 300, 64], nodes=[33, 0, 1, 20], tree=True)
    check_rope(c, ec.rope_inv_freq(hd // 2 * 2, 1e6), 0)
    c["parent"][0] = -1
    check_rope(c, ec.rope_inv_freq(hd // 2 * 2, 1e6), 1)


@pytest.mark.parametrize("H,KVH,hd", [(1, 1, 4), (1, 1, 8), (2, 1, 16), (5, 5, 12), (3, 1, 64), (64, 8, 128)])
def test_rope_narrow_and_wide_rows(H, KVH, hd):
    """Blocks of one wave to four, rows of fewer heads than a block has groups and of
    many more."""
    c = rope_case(8, H, KVH, hd, 3, 9, [10, 0, 300], nodes=[9, 4, 1], tree=True)
    for rot, layout in ((0, 0), (hd // 8 * 8, 0), (hd // 2 * 2, 1), (2, 1)):
        check_rope(c, ec.rope_inv_freq(rot, 1e4) if rot else None, layout)


def test_rope_prompts():
    c = rope_case(7, 14, 2, 64, 2, 700, [0, 33], nodes=[700, 123])
    check_rope(c, ec.rope_inv_freq(64, 1e6))


def test_rope_small_and_large_values():
    c = rope_case(11, 4, 2, 64, 1, 4, [9])
    c["qkv"][0] = 0.0        # eps alone under the root
    c["qkv"][1] *= 1e-20
    c["qkv"][2] *= 1e15
    c["qkv"][3, :64] = 1e-4
    check_rope(c, ec.rope_inv_freq(64, 1e4))


def test_rope_in_place():
    c = rope_case(12, 14, 2, 64, 2, 5, [9, 0])
    inv = ec.rope_inv_freq(64, 1e4)
    want, kw, vw = check_rope(c, inv)
    M, W = c["qkv"].shape
    with ec._Call() as k:
        x, kc, vc = k.put("x", c["qkv"], np.float32), k.put("kc", c["kc"], np.uint16), k.put("vc", c["vc"], np.uint16)
        g = [k.put("qg", c["qg"], np.float32), k.put("kg", c["kg"], np.float32), k.put("f", inv, np.float64)]
        nslots, Cr, _ = c["kc"].shape
        rc = ec.lib().ec_qk_norm_rope_dev(x, W, x, W, kc, vc, nslots, Cr, 14, 2, 64, g[0], g[1], 1e-6, g[2], 64, 0, 1.0,
                                          *k.tree(c["slot"], c["past"], None, None), 2, 5)
        assert rc == 0 and ec.lib().ec_sync() == 0
        got = k.get("x", np.float32, (M, W))
        assert np.array_equal(got[:, :14 * 64], want) and np.array_equal(got[:, 14 * 64:], c["qkv"][:, 14 * 64:])
        assert np.array_equal(k.get("kc", np.uint16, kw.shape), kw) and np.array_equal(k.get("vc", np.uint16, vw.shape), vw)


@pytest.mark.parametrize("name,at,value", BAD)
@pytest.mark.parametrize("hd", [64, 42])
def test_rope_bad_numbers(hd, name, at, value):
    c = rope_case(13, 4, 2, hd, 3, 8, [50, 60, 40], nodes=[8, 7, 8], tree=True, C=100)
    c[name][at] = value
    if name == "nodes":  # all N rows are marked
        q0 = np.full((24, 4 * hd), 7.25, np.float32)
        got, kc, vc = ec.qk_norm_rope_dev(c["qkv"], c["kc"], c["vc"], 4, 2, c["past"], 8, slot=c["slot"], nodes=c["nodes"],
                                          parent=c["parent"], q=q0)
        assert np.isnan(got[8:16]).all() and np.isfinite(got[:8]).all() and np.isfinite(got[16:]).all()
        s = c["slot"][1]
        assert np.array_equal(kc[s], c["kc"][s]) and np.array_equal(vc[s], c["vc"][s])
    else:
        check_rope(c, ec.rope_inv_freq(hd, 1e4), bad=(1,))


def test_rope_same_rows_twice():
    """Of two sequences with a row in common the first writes it; next to each
    other both do."""
    c = rope_case(14, 4, 2, 64, 3, 8, [50, 57, 58], C=100)
    c["slot"][:] = 1
    check_rope(c, ec.rope_inv_freq(64, 1e4), bad=(1, 2))
    c["past"][:] = [50, 58, 42]
    check_rope(c, ec.rope_inv_freq(64, 1e4))


def test_rope_same_rows_as_one_that_writes_none():
    """An earlier sequence with bad parents, or itself too late, still excludes a later
    one; one that names no rows does not."""
    c = rope_case(17, 4, 2, 64, 3, 8, [50, 57, 64], C=100, tree=True)
    c["slot"][:] = 1
    c["parent"][0, 3] = 5
    check_rope(c, ec.rope_inv_freq(64, 1e4), bad=(0, 1, 2))
    c["past"][0] = 93
    check_rope(c, ec.rope_inv_freq(64, 1e4), bad=(0, 2))


def test_rope_same_rows_far_apart():
    """Among 600 sequences: pairs that share a row, next to each other and far apart."""
    c = rope_case(15, 2, 1, 16, 600, 2, [5] * 600)
    for late, early in ((1, 0), (300, 43), (513, 256), (599, 3)):
        c["slot"][late] = c["slot"][early]
    c["past"][513] = 4
    check_rope(c, ec.rope_inv_freq(16, 1e4), bad=(1, 300, 513, 599))


# ---------------------------------------------------------------------------
# accepted rows
# ---------------------------------------------------------------------------

def accept_case(seed, layers, kv, B, N, past, agree=0.8, nodes=None, C=None, vocab=50):
    rng = np.random.default_rng(seed)
    past = np.array(past, np.int32)
    C = C or int(past.max()) + N
    parent = trees(rng, B, N)
    token, sampled = (rng.integers(0, vocab, (B, N)).astype(np.int32) for _ in range(2))
    for b, i in zip(*np.nonzero(rng.random((B, N)) < agree)):
        if i:
            sampled[b, parent[b, i]] = token[b, i]
    shape = (layers, B + 1, C, kv)
    return dict(past=past, parent=parent, token=token, sampled=sampled, kc=rng.integers(0, 65536, shape).astype(np.uint16),
                vc=rng.integers(0, 65536, shape).astype(np.uint16), slot=rng.permutation(B + 1)[:B].astype(np.int32),
                nodes=None if nodes is None else np.array(nodes, np.int32))


def check_accept(c, bad=()):
    B, N = c["token"].shape
    got = ec.tree_accept_dev(c["kc"], c["vc"], c["past"], c["token"], c["sampled"], c["slot"], c["nodes"], c["parent"])
    kw, vw = c["kc"].copy(), c["vc"].copy()
    for b in range(B):
        n = N if c["nodes"] is None else c["nodes"][b]
        line, nxt = [], -1
        if b not in bad and n > 0:
            line = [0]
            while True:
                cur = line[-1]
                nxt = c["sampled"][b, cur]
                kids = [i for i in range(cur + 1, n) if (i - 1 if c["parent"] is None else c["parent"][b, i]) == cur and
                        c["token"][b, i] == nxt and nxt >= 0]
                if not kids:
                    break
                line.append(kids[0])
            p = c["past"][b]
            for cache in (kw, vw):
                cache[:, c["slot"][b], p:p + len(line)] = cache[:, c["slot"][b], [p + j for j in line]].copy()
        assert list(got[0][b]) == line + [-1] * (N - len(line))
        assert (got[1][b], got[2][b], got[3][b]) == (len(line), nxt, c["past"][b] + len(line))
    assert np.array_equal(got[4], kw) and np.array_equal(got[5], vw)
    return got


@pytest.mark.parametrize("layers,kv,B,N,past", [(1, 128, 1, 1, [0]), (24, 128, 1, 8, [700]), (28, 256, 16, 64, range(100, 116)),
                                                (3, 84, 5, 33, [0, 7, 1, 64, 63]), (2, 7, 3, 64, [5, 0, 9]), (2, 768, 4, 5, [3, 2, 1, 0]),
                                                (2, 2050, 2, 20, [3, 2])])
def test_accept_sizes(layers, kv, B, N, past):
    check_accept(accept_case(kv + N, layers, kv, B, N, list(past)))
    check_accept(accept_case(kv + N, layers, kv, B, N, list(past), agree=0.0))


def test_accept_paths():
    """Whole chains, paths that move every row, several children with one token,
    tokens that confirm nothing, padding."""
    c = accept_case(2, 3, 64, 6, 64, [4, 0, 11, 2, 40, 9], nodes=[64, 64, 64, 64, 0, 30], vocab=3)
    c["parent"][0] = np.arange(64) - 1
    c["token"][0], c["sampled"][0] = 5, 5                           # the whole chain
    c["parent"][1] = np.maximum(np.arange(64) - 2, np.where(np.arange(64) == 0, -1, 0))
    c["token"][1], c["sampled"][1] = 5, 5
    c["token"][1, 1] = 6                                            # 0, 2, 4, ...
    c["parent"][2] = np.where(np.arange(64) == 0, -1, 0)
    c["token"][2], c["sampled"][2] = 1, 1                           # of 63 children the first
    c["sampled"][3], c["token"][3] = -1, -1
    got = check_accept(c)
    assert list(got[1]) == [64, 32, 2, 1, 0, got[1][5]]
    c["parent"], c["nodes"] = None, None
    check_accept(c)
    c["slot"] = None
    got = ec.tree_accept_dev(c["kc"], c["vc"], c["past"], c["token"], c["sampled"])
    assert got[1][0] == 64


@pytest.mark.parametrize("name,at,value", BAD)
def test_accept_bad_numbers(name, at, value):
    c = accept_case(13, 2, 64, 3, 8, [50, 60, 40], nodes=[8, 7, 8], C=100)
    c[name][at] = value
    if name in ("past", "nodes"):
        got = ec.tree_accept_dev(c["kc"], c["vc"], c["past"], c["token"], c["sampled"], c["slot"], c["nodes"], c["parent"])
        assert got[1][1] == 0 and got[2][1] == -1 and got[3][1] == c["past"][1] and (got[0][1] == -1).all()
        assert np.array_equal(got[4][:, c["slot"][1]], c["kc"][:, c["slot"][1]]) and got[1][0] > 0 and got[1][2] > 0
    else:
        check_accept(c, bad=(1,))


@pytest.mark.parametrize("kv", [128, 12])
def test_accept_long_moves(kv):
    """Paths of 32 and 63 rows of which every one moves."""
    c = accept_case(21, 2, kv, 2, 64, [7, 30])
    c["parent"][0] = np.maximum(np.arange(64) - 2, np.where(np.arange(64) == 0, -1, 0))
    c["parent"][1] = np.where(np.arange(64) == 2, 0, np.arange(64) - 1)
    c["token"][:], c["sampled"][:] = 5, 5
    c["token"][:, 1] = 6
    got = check_accept(c)
    assert list(got[1]) == [32, 63]


def test_accept_same_rows_twice():
    c = accept_case(14, 2, 64, 3, 8, [50, 57, 58], C=100)
    c["slot"][:] = 1
    check_accept(c, bad=(1, 2))


def test_accept_same_rows_as_one_that_keeps_none():
    """As for the appends: bad parents, too late itself, no rows."""
    c = accept_case(17, 2, 64, 3, 8, [50, 57, 64], C=100)
    c["slot"][:] = 1
    c["parent"][0, 3] = 5
    check_accept(c, bad=(0, 1, 2))
    c["past"][0] = 93
    check_accept(c, bad=(0, 2))


def test_accept_unaligned_rows():
    """Caches at an odd multiple of two bytes."""
    c = accept_case(15, 2, 128, 2, 9, [5, 3])
    want = check_accept(c)
    with ec._Call() as k:
        for n in ("kc", "vc"):
            k.put(n, np.concatenate([np.zeros(1, np.uint16), c[n].ravel()]), np.uint16)
        t = [k.put("token", c["token"], np.int32), k.put("sampled", c["sampled"], np.int32)]
        o = [k.put(n, np.zeros(s), np.int32) for n, s in (("path", 18), ("npath", 2), ("next", 2), ("new_past", 2))]
        layers, nslots, Cr, kv = c["kc"].shape
        rc = ec.lib().ec_tree_accept_dev(k.ptr("kc") + 2, k.ptr("vc") + 2, layers, nslots, Cr, kv,
                                         *k.tree(c["slot"], c["past"], None, c["parent"]), *t, 2, 9, *o)
        assert rc == 0 and ec.lib().ec_sync() == 0
        for n, w in (("kc", want[4]), ("vc", want[5])):
            assert np.array_equal(k.get(n, np.uint16, c[n].size + 1)[1:], w.ravel())


@pytest.mark.parametrize("layers,kv,B,N", [(1, 1, 3, 4), (3, 7, 2, 64), (2, 8, 1, 2), (5, 520, 2, 9)])
def test_accept_narrow_rows(layers, kv, B, N):
    check_accept(accept_case(kv, layers, kv, B, N, range(3, 3 + B)))


# ---------------------------------------------------------------------------
# the largest batch, and arguments that may be missing
# ---------------------------------------------------------------------------

def test_largest_batch():
    """65535 sequences of 64 rows through all of the cache's operators, checked at
    the ends and in between."""
    B, N, hd, Cr = 65535, 64, 4, 70
    rng = np.random.default_rng(77)
    x = rng.normal(0, 2, (B * N, 3 * hd)).astype(np.float32)
    past = rng.integers(0, Cr - N + 1, B).astype(np.int32)
    at = [0, 1, 255, 256, 32767, 32768, B - 2, B - 1]
    kc = np.zeros((B, Cr, hd), np.uint16)
    inv = ec.rope_inv_freq(hd, 1e4)
    q, k, v = ec.qk_norm_rope_dev(x, kc, kc, 1, 1, past, N, inv_freq=inv)
    for b in at:
        one = ec.qk_norm_rope_dev(x[b * N:(b + 1) * N], kc[b:b + 1], kc[b:b + 1], 1, 1, past[b:b + 1], N, inv_freq=inv)
        assert np.array_equal(q[b * N:(b + 1) * N], one[0])
        assert np.array_equal(k[b], one[1][0]) and np.array_equal(v[b], one[2][0])
    att = ec.attention_tree_dev(q, k, v, 1, 1, past, N)
    for b in at:
        check_attention(dict(H=1, KVH=1, past=past[b:b + 1], N=N, q=q[b * N:(b + 1) * N], kc=k[b:b + 1], vc=v[b:b + 1],
                             slot=None, parent=None, nodes=None), got=att[b * N:(b + 1) * N])
    token = rng.integers(0, 3, (B, N)).astype(np.int32)
    path, npath, nxt, new, k2, _ = ec.tree_accept_dev(k[None], v[None], past, token, np.roll(token, -1, 1))
    # a chain whose sampled tokens are the next node's: all of it stays but for what
    # the last one's says
    assert (npath == N).all() and (path == np.arange(N)).all() and np.array_equal(new, past + N)
    assert np.array_equal(nxt, token[:, 0]) and np.array_equal(k2[0], k)


def test_largest_batch_on_the_matrix_cores():
    """As many rows for the form of tiles, one KV head of 32."""
    B, N, hd, Cr = 65535, 64, 32, 65
    rng = np.random.default_rng(78)
    q = np.tile(rng.normal(0, 1, (N * 5, hd)).astype(np.float32), (B // 5, 1))
    kc, vc = (f16(rng.normal(0, 1, (7, Cr, hd))) for _ in range(2))
    slot, past = (np.arange(B) % 7).astype(np.int32), (np.arange(B) % 2).astype(np.int32)
    got = ec.attention_tree_dev(q, kc, vc, 1, 1, past, N, slot)
    for b in (0, 1, 4097, 32768, B - 1):
        check_attention(dict(H=1, KVH=1, past=past[b:b + 1], N=N, q=q[b * N:(b + 1) * N], kc=kc, vc=vc, slot=slot[b:b + 1],
                             parent=None, nodes=None), got=got[b * N:(b + 1) * N])
    # equal inputs, equal outputs, all through the batch
    assert np.array_equal(got[:70 * N], got[65450 * N:65520 * N])


def test_more_blocks_than_a_grid_dimension():
    """65535 one-token sequences of 260 heads: blocks of 256 threads that are more than
    2^32 threads in all."""
    B, H, hd = 65535, 260, 32
    assert B * H * 256 > 2 ** 32
    rng = np.random.default_rng(79)
    few = rng.normal(0, 1, (15, H * hd)).astype(np.float32)
    kc, vc = (f16(rng.normal(0, 1, (7, 3, H * hd))) for _ in range(2))
    slot, past = (np.arange(B) % 7).astype(np.int32), (np.arange(B) % 3).astype(np.int32)
    got = ec.attention_tree_dev(np.tile(few, (B // 15, 1)), kc, vc, H, H, past, 1, slot, max_past=2)
    for b in (0, 1, 32768, 65011, B - 2, B - 1):
        check_attention(dict(H=H, KVH=H, past=past[b:b + 1], N=1, q=few[b % 15:b % 15 + 1], kc=kc, vc=vc, slot=slot[b:b + 1],
                             parent=None, nodes=None), got=got[b:b + 1])
    # equal inputs every 105 sequences, equal outputs all through the batch
    assert np.array_equal(got[:-105], got[105:])


def test_one_norm_alone():
    for name in ("qg", "kg"):
        for hd in (64, 42):
            c = rope_case(16, 4, 2, hd, 2, 3, [7, 0])
            c[name] = None
            check_rope(c, ec.rope_inv_freq(hd // 2 * 2, 1e4))


def test_sample_without_probabilities():
    rng = np.random.default_rng(18)
    x, u = rng.normal(0, 2, (3, 700)).astype(np.float32), rng.random(3)
    want, _ = ec.sample_dev(x, u)
    with ec._Call() as k:
        p = k.put("x", x, np.float32), k.put("u", u, np.float64), k.put("t", np.zeros(3), np.int32)
        assert ec.lib().ec_sample_dev(p[0], 3, 700, 700, None, None, None, None, p[1], p[2], None) == 0
        assert ec.lib().ec_sync() == 0
        assert np.array_equal(k.get("t", np.int32, 3), want)


def test_shared_slot():
    """Two sequences that read one slot, at lengths of their own."""
    c = attn_case(23, 6, 2, 64, 3, 1, [500, 90, 333], C=600)
    c["slot"][:] = 2
    check_attention(c)


# ---------------------------------------------------------------------------
# together
# ---------------------------------------------------------------------------

class _Step:
    """One checking step of one layer on device buffers: rows -> cache, tree
    attention, a language-model head, sampling, what stays."""
    H, KVH, hd, V, B, N, C, layers = 6, 2, 64, 501, 3, 8, 160, 1

    def __init__(self, seed):
        r = self.rng = np.random.default_rng(seed)
        s, E = self, self.H * self.hd
        self.k = k = ec._Call()
        s.head = (r.normal(0, 0.06, (s.V, E))).astype(np.float16)
        s.qg, s.kg = (r.normal(1, 0.2, s.hd).astype(np.float32) for _ in range(2))
        s.inv = ec.rope_inv_freq(s.hd, 1e4)
        cache = [f16(r.normal(0, 1, (s.B, s.C, s.KVH * s.hd))) for _ in range(2)]
        M = s.B * s.N
        for n, a, t in (("head", s.head.view(np.uint16), np.uint16), ("qg", s.qg, np.float32), ("kg", s.kg, np.float32),
                        ("inv", s.inv, np.float64), ("kc", cache[0], np.uint16), ("vc", cache[1], np.uint16),
                        ("slot", [2, 0, 1], np.int32), ("temp", [0.0] * M, np.float32),
                        ("q", np.zeros((M, E)), np.float32), ("att", np.zeros((M, E)), np.float32),
                        ("logits", np.zeros((M, s.V)), np.float32), ("sampled", np.zeros(M), np.int32),
                        ("prob", np.zeros(M), np.float32), ("path", np.zeros(M), np.int32), ("npath", np.zeros(s.B), np.int32),
                        ("next", np.zeros(s.B), np.int32), ("new_past", np.zeros(s.B), np.int32),
                        ("x", np.zeros((M, (s.H + 2 * s.KVH) * s.hd)), np.float32), ("past", np.zeros(s.B), np.int32),
                        ("nodes", np.zeros(s.B), np.int32), ("parent", np.zeros(M), np.int32),
                        ("token", np.zeros(M), np.int32), ("u", np.zeros(M), np.float64)):
            k.put(n, a, t)

    def new(self):
        """New inputs in the same buffers."""
        s, r, M = self, self.rng, self.B * self.N
        s.x = r.normal(0, 2, (M, (s.H + 2 * s.KVH) * s.hd)).astype(np.float32)
        s.past = r.integers(0, s.C - s.N + 1, s.B).astype(np.int32)
        s.nodes = r.integers(1, s.N + 1, s.B).astype(np.int32)
        s.parent = trees(r, s.B, s.N, 2)
        s.token, s.u = r.integers(0, s.V, (s.B, s.N)).astype(np.int32), r.random(M)
        s.temp = np.where(r.random(M) < 0.3, 0.0, 0.7).astype(np.float32)
        for n in ("x", "past", "nodes", "parent", "token", "u", "temp"):
            a = np.ascontiguousarray(getattr(s, n))
            assert ec.lib().ec_memcpy_h2d(s.k.ptr(n), a.ctypes.data, a.nbytes) == 0

    def call(self):
        s, L, p = self, ec.lib(), self.k.ptr
        E, W, M = s.H * s.hd, (s.H + 2 * s.KVH) * s.hd, s.B * s.N
        tree = (p("slot"), p("past"), p("nodes"), p("parent"))
        return (L.ec_qk_norm_rope_dev(p("x"), W, p("q"), E, p("kc"), p("vc"), s.B, s.C, s.H, s.KVH, s.hd, p("qg"), p("kg"),
                                      1e-6, p("inv"), s.hd, 0, 1.0, *tree, s.B, s.N)
                or L.ec_attention_tree_dev(p("q"), E, p("kc"), p("vc"), s.B, s.C, s.H, s.KVH, s.hd, *tree, s.B, s.N, s.C, 0,
                                           p("att"), E)
                or L.ec_gemm_fp16_fp32_dev(p("logits"), p("att"), p("head"), M, E, s.V)
                or L.ec_sample_dev(p("logits"), M, s.V, s.V, p("temp"), None, None, None, p("u"), p("sampled"), p("prob"))
                or L.ec_tree_accept_dev(p("kc"), p("vc"), 1, s.B, s.C, s.KVH * s.hd, *tree, p("token"), p("sampled"), s.B,
                                        s.N, p("path"), p("npath"), p("next"), p("new_past")))

    def caches(self):
        return [self.k.get(n, np.uint16, (self.B, self.C, self.KVH * self.hd)) for n in ("kc", "vc")]

    def outputs(self):
        s, M = self, self.B * self.N
        g = s.k.get
        return [g("q", np.uint32, M * s.H * s.hd), g("att", np.uint32, M * s.H * s.hd), g("sampled", np.int32, M),
                g("path", np.int32, M), g("npath", np.int32, s.B), g("next", np.int32, s.B), g("new_past", np.int32, s.B),
                *s.caches()]


def test_step_together():
    """The operators in a row against the plain ones in a row, each on the
    device's own input to it."""
    s = _Step(1)
    try:
        for _ in range(3):
            s.new()
            before = s.caches()
            assert s.call() == 0, ec.last_error()
            assert ec.lib().ec_sync() == 0
            B, N, H, KVH, hd = s.B, s.N, s.H, s.KVH, s.hd
            slot = np.array([2, 0, 1], np.int32)
            q, kc, vc = ec.qk_norm_rope_dev(s.x, *before, H, KVH, s.past, N, s.qg, s.kg, 1e-6, s.inv, slot=slot,
                                            nodes=s.nodes, parent=s.parent, q=s.k.get("q", np.float32, (B * N, H * hd)))
            att = s.k.get("att", np.float32, (B * N, H * hd))
            live = np.repeat(np.arange(N)[None], B, 0) < s.nodes[:, None]
            case = dict(H=H, KVH=KVH, past=s.past, N=N, q=q, kc=kc, vc=vc, slot=slot, parent=s.parent, nodes=s.nodes)
            check_attention(case, got=np.where(live.reshape(-1, 1), att, np.float32(7.25)))
            logits = s.k.get("logits", np.float32, (B * N, s.V))
            want = att[live.ravel()].astype(np.float64) @ s.head.T.astype(np.float64)
            assert np.abs(logits[live.ravel()] - want).max() < 1e-4
            sampled = s.k.get("sampled", np.int32, (B, N))
            for m in range(B * N):
                assert sampled.ravel()[m] == ref_sample(logits[m], s.u[m], s.temp[m])[0]
            got = s.k.get("path", np.int32, (B, N)), *(s.k.get(n, np.int32, B) for n in ("npath", "next", "new_past"))
            again = ec.tree_accept_dev(kc[None], vc[None], s.past, s.token, sampled, slot, s.nodes, s.parent)
            for a, b in zip(got, again):
                assert np.array_equal(a, b)
            for a, b in zip(s.caches(), again[4:]):
                assert np.array_equal(a, b[0])
    finally:
        s.k.__exit__()


class _Graph:
    """What `call` enqueues on ec_stream(), captured."""

    def __init__(self, call):
        self.hip = C.CDLL("libamdhip64.so")
        self.stream = C.c_void_p(ec.lib().ec_stream())
        graph, self.exec = C.c_void_p(), C.c_void_p()
        assert self.hip.hipStreamBeginCapture(self.stream, 1) == 0  # thread-local
        rc, err = call(), ec.last_error()
        assert self.hip.hipStreamEndCapture(self.stream, C.byref(graph)) == 0
        assert rc == 0, err
        assert self.hip.hipGraphInstantiate(C.byref(self.exec), graph, None, None, C.c_size_t(0)) == 0
        assert self.hip.hipGraphDestroy(graph) == 0

    def replay(self):
        assert self.hip.hipGraphLaunch(self.exec, self.stream) == 0

    def close(self):
        assert self.hip.hipGraphExecDestroy(self.exec) == 0


def test_step_captured():
    """Two steps' graphs (they share the library's workspace), replayed in turn
    with new inputs, eager calls and larger ones between: the eager results."""
    L = ec.lib()
    a, b = _Step(2), _Step(3)
    big = attn_case(50, 12, 2, 128, 4, 16, [6000, 10, 3000, 5])
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
                kept = s.caches()
                assert s.call() == 0 and L.ec_sync() == 0
                want.append(s.outputs())
                for n, c in zip(("kc", "vc"), kept):
                    assert L.ec_memcpy_h2d(s.k.ptr(n), c.ctypes.data, c.nbytes) == 0
            graphs[turn % 2].replay()
            graphs[1 - turn % 2].replay()
            assert L.ec_sync() == 0
            for s, w in zip((a, b), want):
                for x, y in zip(s.outputs(), w):
                    assert np.array_equal(x, y)
            check_attention(big, rows=[(0, 3), (2, 15)])
    finally:
        for g in graphs:
            g.close()
        a.k.__exit__()
        b.k.__exit__()


def test_release_between():
    """The workspace goes with ec_release; the next call makes a new one."""
    c = attn_case(51, 12, 2, 128, 2, 4, [900, 100])
    first = check_attention(c)
    assert ec.lib().ec_release() == 0 or "models still loaded" in ec.last_error()
    assert np.array_equal(check_attention(c), first)


def test_capture_without_a_workspace():
    """A captured call whose workspace is not there yet is refused, the capture ends as
    ever, and the same call runs after an eager one has made it."""
    L = ec.lib()
    if L.ec_release():
        pytest.skip("models are loaded")
    c = attn_case(52, 12, 2, 128, 2, 4, [900, 100])
    rng = np.random.default_rng(53)
    x, u = rng.normal(0, 2, (3, 5000)).astype(np.float32), rng.random(3)
    nslots, Cr, _ = c["kc"].shape
    E = 12 * 128
    with ec._Call() as k:
        a = [k.put("q", c["q"], np.float32), E, k.put("kc", c["kc"], np.uint16), k.put("vc", c["vc"], np.uint16), nslots, Cr, 12, 2,
             128, *k.tree(c["slot"], c["past"], None, c["parent"]), 2, 4, Cr, 0, k.put("out", np.zeros_like(c["q"]), np.float32), E]
        b = [k.put("x", x, np.float32), 3, 5000, 5000, None, None, None, None, k.put("u", u, np.float64),
             k.put("token", np.zeros(3), np.int32), None]
        for call, read in ((lambda: L.ec_attention_tree_dev(*a), lambda: k.get("out", np.float32, c["q"].shape)),
                           (lambda: L.ec_sample_dev(*b), lambda: k.get("token", np.int32, 3))):
            before = read()
            with pytest.raises(AssertionError, match="inside a stream capture"):
                _Graph(call)
            assert np.array_equal(read(), before)
            assert call() == 0 and L.ec_sync() == 0
            want = read()
            g = _Graph(call)
            for _ in range(3):
                g.replay()
                assert L.ec_sync() == 0 and np.array_equal(read(), want)
            g.close()
        check_attention(c, got=k.get("out", np.float32, c["q"].shape))
        assert [ref_sample(x[r], u[r])[0] for r in range(3)] == list(k.get("token", np.int32, 3))


def test_profiled_calls():
    """The calls under the library's per-kernel timing."""
    import json
    s = _Step(4)
    L = ec.lib()
    try:
        s.new()
        assert L.ec_prof_start(b"") == 0 and s.call() == 0
        buf = C.create_string_buffer(1 << 16)
        assert L.ec_prof_stop(buf, len(buf)) > 0
        names = {r["kernel"] for r in json.loads(buf.value.decode())}
        assert {"qk_norm_rope", "attention_tree", "attention_tree_join", "sample_top", "sample_bins", "sample_pick",
                "tree_accept"} <= names
    finally:
        s.k.__exit__()
