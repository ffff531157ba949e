"""Captured calls over a paged cache do the work themselves: everything that a replay
writes holds something else before it."""
import ctypes as C

import numpy as np
import pytest

import edgecore_amd as ec
from test_gpu_paged_ops import _Serve, attn_case, check
from test_gpu_tree_ops import _Graph

pytestmark = pytest.mark.gpu

L = None


@pytest.fixture(autouse=True)
def _lib():
    global L
    L = ec.lib()


def fill(k, names):
    """Bytes of 0xA5 (as fp32 and fp16 small negative numbers, as a token none)."""
    for n in names:
        b = k.bufs[n]
        assert L.ec_memset_dev(b.ptr, 0xA5, b.nbytes) == 0


OUTPUTS = ("q", "att", "logits", "edited", "token", "kc", "vc")


def reset(s, pages):
    """Outputs that hold something else, pages as they were."""
    fill(s.k, OUTPUTS)
    for n in ("k", "v", "k_scale", "v_scale"):
        a = getattr(pages, n)
        if a is not None:
            assert L.ec_memcpy_h2d(s.k.ptr("pages." + n), a.ctypes.data, a.nbytes) == 0
    assert L.ec_sync() == 0


def everything(s):
    """The bytes of all that a call may write, padding included."""
    raw = [s.k.get(n, np.uint8, s.k.bufs[n].nbytes) for n in OUTPUTS]
    now = s.pages.got(s.k)
    return raw + [getattr(now, n) for n in ("k", "v", "k_scale", "v_scale") if getattr(now, n) is not None]


@pytest.mark.parametrize("first", ["eager", "replay"])
@pytest.mark.parametrize("types", [("int8", "fp16"), ("e4m3", "int8")])
def test_replays_do_the_work(first, types):
    """Graphs of single tokens and of chunks (they share the library's workspace), replayed in
    turn with new inputs, from cleared outputs and from the pages that the eager calls started with;
    eager calls and larger ones between.  The eager call comes before the replay, or after it."""
    a, b = _Serve(2, types[0], 5, 1), _Serve(3, types[1], 90, 0)
    big = attn_case(50, "e4m3", 12, 2, 128, 16, [6000, 10, 3000], [40, 200, 1])
    graphs = []

    def eager():
        got = []
        for s, pages in zip((a, b), before):
            reset(s, pages)
            assert s.call() == 0, ec.last_error()
            assert L.ec_sync() == 0
            got.append(everything(s))
        return got

    def replayed(order):
        for s, pages in zip((a, b), before):
            reset(s, pages)
        for i in order:
            graphs[i].replay()
        assert L.ec_sync() == 0
        return [everything(s) for s in (a, b)]

    try:
        for s in (a, b):
            s.new()
            assert s.call() == 0 and L.ec_sync() == 0
        graphs = [_Graph(a.call), _Graph(b.call)]
        for turn in range(4):
            for s in (a, b):
                s.new()
            before = [s.pages.got(s.k) for s in (a, b)]
            order = (turn % 2, 1 - turn % 2)
            got = [eager(), replayed(order)] if first == "eager" else [replayed(order), eager()]
            for want, have in zip(*got):
                for x, y in zip(want, have):
                    assert np.array_equal(x, y)
                # and they are not what they were filled with
                assert not (want[OUTPUTS.index("att")] == 0xA5).all() and not (want[OUTPUTS.index("kc")] == 0xA5).all()
            for s, w in zip((a, b), got[0]):
                for n in ("q", "att", "edited", "token"):
                    rows = w[OUTPUTS.index(n)].reshape(s.M, -1)
                    assert (rows[s.start[-1]:] == 0xA5).all() or n in ("edited", "token")  # rows of no sequence
                    assert not (rows[:s.start[-1]] == 0xA5).all(1).any()
            check(big, rows=[(0, 3), (1, 150), (2, 0)])
    finally:
        for g in graphs:
            g.close()
        a.k.__exit__()
        b.k.__exit__()


@pytest.mark.parametrize("new", [[1, 1], [200, 3]])
def test_replay_with_a_workspace_of_its_own(new):
    """A graph keeps the workspace that it was captured with, also when a larger call has
    made another: each replay writes every row anew, in parts that are joined."""
    c = attn_case(13, "int8", 12, 2, 128, 16, [3000, 100], new, pad=0)
    E, M = 12 * 128, sum(new)
    with ec._Call() as k:
        cache = c["pages"].put(k)
        a = [C.byref(cache), k.put("q", c["q"], np.float32), E, 12, k.put("start", c["start"], np.int32),
             k.put("past", c["past"], np.int32), 2, M, 3000, 0, 0, k.put("out", np.full_like(c["q"], 7.25), np.float32), E]
        read = lambda: k.get("out", np.float32, c["q"].shape)  # noqa: E731
        run = lambda: L.ec_attention_paged_dev(*a)  # noqa: E731
        assert run() == 0 and L.ec_sync() == 0
        want = read()
        check(c, got=np.concatenate((want, np.full((1, E), 7.25, np.float32))), rows=[(0, 0), (0, new[0] - 1), (1, 0)])
        g = _Graph(run)
        for larger in (0, 9000, 30000):
            if larger:
                check(attn_case(14, "fp16", 12, 2, 128, 16, [larger, 8000], [300, 200]), rows=[(0, 299), (1, 0)])
            for _ in range(3):
                fill(k, ["out"])
                assert L.ec_sync() == 0
                g.replay()
                assert L.ec_sync() == 0 and np.array_equal(read(), want)
        g.close()
