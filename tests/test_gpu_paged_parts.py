"""Attention over a paged cache in parts that are joined: with the output in place of the
queries, and with starts that do not ascend, behind a call that left other rows' places in the
workspace.  That a call is joined is read from the library's timing."""
import ctypes as C
import json

import numpy as np
import pytest

import edgecore_amd as ec
from test_gpu_paged_ops import attn_case, check

pytestmark = pytest.mark.gpu


def kernels(run):
    """What `run` launches."""
    L = ec.lib()
    assert L.ec_prof_start(b"") == 0
    try:
        assert run() == 0, ec.last_error()
    finally:
        buf = C.create_string_buffer(1 << 16)
        n = L.ec_prof_stop(buf, len(buf))
    assert n > 0
    return {r["kernel"] for r in json.loads(buf.value.decode())}


def attend(c, window=0, sinks=0, in_place=False):
    """(out, kernels) of a call whose rows have others in front of and behind them."""
    pages, H = c["pages"], c["H"]
    M, E = c["q"].shape
    guard = 8
    with ec._Call() as k:
        def rows(a):
            x = np.full((M + 2 * guard, E), 7.25, np.float32)
            x[guard:guard + M] = a
            return x

        cache = pages.put(k)
        q = k.put("q", rows(c["q"]), np.float32) + 4 * guard * E
        o = q if in_place else k.put("o", rows(7.25), np.float32) + 4 * guard * E
        start, past = k.put("start", c["start"], np.int32), k.put("past", c["past"], np.int32)
        names = kernels(lambda: ec.lib().ec_attention_paged_dev(C.byref(cache), q, E, H, start, past, len(c["past"]), M,
                                                                int(c["past"].max()), window, sinks, o, E))
        got = k.get("q" if in_place else "o", np.float32, (M + 2 * guard, E))
        now = pages.got(k)
    for n in ("k", "v", "k_scale", "v_scale"):
        a = getattr(pages, n)
        assert a is None or np.array_equal(a, getattr(now, n))
    assert (got[:guard] == 7.25).all() and (got[guard + M:] == 7.25).all()
    return got[guard:guard + M], names


SHAPES = [("e4m3", 14, 2, 64), ("int8", 12, 2, 128), ("fp16", 16, 4, 96), ("int8", 8, 1, 32)]


@pytest.mark.parametrize("type,H,KVH,hd", SHAPES)
@pytest.mark.parametrize("past,new", [([3000, 40], [1, 1]), ([3000, 2500, 17], [150, 1, 9]), ([0, 900], [1200, 300])])
@pytest.mark.parametrize("window,sinks", [(0, 0), (700, 4)])
def test_in_place(type, H, KVH, hd, past, new, window, sinks):
    c = attn_case(hd + new[0], type, H, KVH, hd, 16, past, new, pad=1)
    want, names = attend(c, window, sinks)
    live = c["start"][-1]
    # (single tokens of narrow heads see too little through the window to be in parts)
    assert ("attention_paged_join" in names) == (max(new) > 1 or not window or hd > 64)
    some = {(b, i) for b, n in enumerate(new) for i in {0, n // 2, n - 1}}
    check(c, window, sinks, rows=some, got=want)
    got, _ = attend(c, window, sinks, in_place=True)
    assert np.array_equal(got[:live], want[:live]) and np.array_equal(got[live:], c["q"][live:])


# of 300 rows; by those that ascend and stay inside every row is said
STARTS = [[0, 120, 60, 300], [300, 200, 100, 0], [-7, 200, 200, 299], [0, 2 ** 31 - 1, 5, 300], [-2 ** 31, 2 ** 31 - 1, 0, 4],
          [0, 300, 0, 300], [0, 140, 141, 345], [0, 120, 130, 301], [2, 200, 200, 290], [17, 17, 217, 217], [300, 300, 300, 300],
          [0, 0, 0, 300], [5, 6, 7, 8]]


@pytest.mark.parametrize("H,KVH,hd,type", [(4, 2, 64, "int8"), (6, 3, 128, "fp16")])
@pytest.mark.parametrize("start", STARTS)
def test_odd_starts_of_chunks(H, KVH, hd, type, start):
    c = attn_case(33, type, H, KVH, hd, 16, [3000, 2000, 2500], [300, 300, 300], pad=0)
    c["q"] = c["q"][:300]
    run_odd(c, start, 300)


@pytest.mark.parametrize("H,KVH,hd,type", [(4, 2, 64, "int8"), (6, 3, 128, "fp16")])
@pytest.mark.parametrize("start", [[0, 5, 3, 9], [9, 6, 3, 0], [-7, 2, 2, 9], [0, 2 ** 31 - 1, 5, 9], [0, 9, 0, 9], [0, 4, 5, 12],
                                   [2, 4, 4, 5], [1, 1, 1, 9], [9, 9, 9, 9]])
def test_odd_starts_of_few_rows(H, KVH, hd, type, start):
    c = attn_case(34, type, H, KVH, hd, 16, [3000, 2000, 2500], [9, 9, 9], pad=0)
    c["q"] = c["q"][:9]
    run_odd(c, start, 9)


def run_odd(c, start, M):
    """In front of it a larger call in parts, whose rows' places the workspace still has."""
    H, E = c["H"], c["q"].shape[1]
    big = attn_case(35, "e4m3", 12, 2, 128, 16, [6000, 5000], [400, 200])
    _, names = attend(big)
    assert "attention_paged_join" in names
    c["start"] = np.array(start, np.int32)
    got, names = attend(c)
    assert "attention_paged_join" in names
    if not all(0 <= a <= b <= M for a, b in zip(start, start[1:])):
        return
    c["new"] = np.diff(c["start"])
    assert (got[:start[0]] == 7.25).all() and (got[start[-1]:] == 7.25).all()
    some = {(b, i) for b, n in enumerate(c["new"]) for i in {0, n // 2, n - 1} if n}
    check(c, rows=some, got=got)
