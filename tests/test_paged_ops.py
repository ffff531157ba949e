"""The operators over a paged cache and the edits of logits without a GPU: what their
entry points refuse (arguments are checked before the device is opened), and the checks
that the kernels make of device arrays (ec_pages.h, compiled for the host)."""
import ctypes as C
import math
import subprocess

import numpy as np
import pytest

import edgecore_amd as ec
from test_tree_ops import refused

REPO = ec.PKG_DIR.parent
P = 1 << 12  # stands for a device pointer: refused calls do not look at it


def cache(**k):
    a = dict(k=1 << 32, v=1 << 33, k_scale=1 << 34, v_scale=1 << 35, type=1, npages=10, page=16, KVH=1, hd=64, table=1 << 20, ldt=4)
    a.update({n: k[n] for n in a if n in k})
    return C.byref(ec.PagedCache(*a.values())) if "cache" not in k else k["cache"]


def fill(a, k):
    assert all(n in a or n in ("k", "v", "k_scale", "v_scale", "type", "npages", "page", "KVH", "hd", "table", "ldt") for n in k)
    a.update({n: v for n, v in k.items() if n in a})
    return a


def append(**k):
    a = fill(dict(cache=None, qkv=P, ldx=4 * 64, q=1 << 17, ldq=128, H=2, qg=None, kg=None, eps=1e-6, inv_freq=P, rot=64, layout=0,
                  factor=1.0, start=1 << 21, past=1 << 22, B=2, M=6), k)
    a["cache"] = cache(**k)
    return ec.lib().ec_paged_append_dev(*a.values())


def attention(**k):
    a = fill(dict(cache=None, q=P, ldq=128, H=2, start=1 << 21, past=1 << 22, B=2, M=6, max_past=50, window=0, sinks=0, out=1 << 17,
                  ldo=128), k)
    a["cache"] = cache(**k)
    return ec.lib().ec_attention_paged_dev(*a.values())


def read(**k):
    a = fill(dict(cache=None, first=1 << 21, count=1 << 22, B=2, max_count=40, kc=1 << 36, vc=1 << 37, nslots=2, C=100, slot=None,
                  to=None), k)
    a["cache"] = cache(**k)
    return ec.lib().ec_paged_read_dev(*a.values())


def edit(**k):
    a = fill(dict(logits=P, ld=100, out=1 << 17, ldo=100, vocab=100, text=1 << 20, ldt=30, len=1 << 21, prompt=None, token=None,
                  nodes=None, parent=None, B=2, N=3, repetition=None, frequency=None, presence=None, bias_token=None, bias=None,
                  nbias=None, max_bias=0, mask=None, ldm=4), k)
    return ec.lib().ec_logits_edit_dev(*a.values())


CACHE = [dict(cache=None), dict(type=-1), dict(type=3), dict(npages=0), dict(npages=-1), dict(page=0), dict(KVH=0), dict(hd=0),
         dict(hd=513, ldx=1 << 20, ldq=1 << 20, ldo=1 << 20), dict(ldt=0), dict(npages=1 << 20, page=1 << 11), dict(k=None),
         dict(v=None), dict(table=None), dict(k_scale=None), dict(type=2, v_scale=None), dict(npages=2 ** 31 - 1, page=2 ** 31 - 1)]
BATCH = [dict(B=0), dict(B=-1), dict(B=65536), dict(past=None), dict(M=0), dict(M=(1 << 22) + 1), dict(start=None)]


def for_(k, *names):
    return {n: v for n, v in k.items() if n not in ("ldx", "ldq", "ldo") or n in names}


@pytest.mark.parametrize("k", [for_(k, "ldx", "ldq") for k in CACHE] + BATCH + [
    dict(H=0), dict(H=3, KVH=2), dict(H=65536, ldx=1 << 30, ldq=1 << 30), dict(ldx=255), dict(ldq=127), dict(rot=63), dict(rot=66),
    dict(rot=-2), dict(layout=2), dict(layout=-1), dict(eps=-1e-6), dict(eps=math.nan), dict(qkv=None), dict(q=None),
    dict(inv_freq=None), dict(q=P), dict(q=P + 256, ldq=256)])
def test_append_refuses(k):
    refused(append(**k), "ec_paged_append_dev")


@pytest.mark.parametrize("k", [for_(k, "ldq", "ldo") for k in CACHE] + BATCH + [
    dict(H=0), dict(H=3, KVH=2), dict(ldq=127), dict(ldo=127), dict(window=-1), dict(sinks=-1), dict(max_past=-1), dict(max_past=65),
    dict(q=None), dict(out=None), dict(out=P, ldo=256), dict(out=P + 512)])
def test_attention_refuses(k):
    refused(attention(**k), "ec_attention_paged_dev")


@pytest.mark.parametrize("k", [for_(k) for k in CACHE] + [
    dict(B=0), dict(B=65536), dict(first=None), dict(count=None), dict(kc=None), dict(vc=None), dict(max_count=0), dict(max_count=-1),
    dict(max_count=(1 << 30) + 1), dict(nslots=0), dict(C=0), dict(C=(1 << 30) + 1)])
def test_read_refuses(k):
    refused(read(**k), "ec_paged_read_dev")


@pytest.mark.parametrize("k", [
    dict(B=0), dict(N=0), dict(B=65536), dict(N=65536), dict(B=65535, N=65), dict(token=P, N=65), dict(vocab=0),
    dict(vocab=(1 << 18) + 1, ld=1 << 19, ldo=1 << 19), dict(ld=99), dict(ldo=99), dict(mask=1 << 22, ldm=3), dict(ldt=-1),
    dict(ldt=(1 << 30) + 1), dict(max_bias=-1), dict(logits=None), dict(out=None), dict(text=None), dict(len=None),
    dict(max_bias=3, bias=P), dict(max_bias=3, bias_token=P), dict(out=P, ldo=128), dict(out=P + 400)])
def test_edit_refuses(k):
    refused(edit(**k), "ec_logits_edit_dev")


N8 = 10 * 16 * 64  # bytes of an int8 cache of cache()


@pytest.mark.parametrize("k", [
    dict(v=1 << 32), dict(v=(1 << 32) + N8 - 1), dict(type=0, v=(1 << 32) + 2 * N8 - 1), dict(k_scale=(1 << 33) + N8 - 1),
    dict(v_scale=(1 << 34) + 2 * 160 - 1), dict(q=(1 << 32) + N8 - 4), dict(qkv=(1 << 33) - 4 * (5 * 256 + 256) + 4),
    dict(table=(1 << 17) + 8), dict(start=1 << 17), dict(past=(1 << 34) + 8), dict(qg=1 << 17), dict(kg=(1 << 35) + 16),
    dict(inv_freq=(1 << 32) - 252), dict(start=(1 << 17) - 8), dict(table=(1 << 17) - 28)])
def test_append_refuses_overlaps(k):
    refused(append(**k), "ec_paged_append_dev", "overlaps")


@pytest.mark.parametrize("k", [
    dict(out=(1 << 32) + N8 - 4), dict(out=(1 << 33) - 4 * (5 * 128 + 128) + 4), dict(out=(1 << 34) + 316), dict(out=1 << 35),
    dict(table=(1 << 17) + 8), dict(start=(1 << 17) - 8), dict(past=1 << 17)])
def test_attention_refuses_overlaps(k):
    refused(attention(**k), "ec_attention_paged_dev", "overlaps another array")


@pytest.mark.parametrize("k", [
    dict(kc=1 << 37), dict(vc=(1 << 36) + 2 * 200 * 64 - 2), dict(kc=(1 << 32) + N8 - 2), dict(vc=1 << 34), dict(table=1 << 36),
    dict(first=1 << 36), dict(count=(1 << 37) - 4), dict(slot=1 << 37), dict(to=(1 << 36) + 100)])
def test_read_refuses_overlaps(k):
    refused(read(**k), "ec_paged_read_dev", "overlaps another array")


@pytest.mark.parametrize("k", [
    dict(text=(1 << 17) - 4 * 60 + 4), dict(len=1 << 17), dict(prompt=(1 << 17) + 2396), dict(token=1 << 17), dict(nodes=1 << 17),
    dict(parent=(1 << 17) - 20), dict(repetition=1 << 17), dict(frequency=1 << 17), dict(presence=1 << 17),
    dict(max_bias=5, bias=1 << 17, bias_token=P), dict(max_bias=5, bias_token=(1 << 17) - 36, bias=P), dict(nbias=(1 << 17) - 4),
    dict(mask=(1 << 17) - 4 * 24 + 4)])
def test_edit_refuses_overlaps(k):
    refused(edit(**k), "ec_logits_edit_dev", "overlaps another array")


def test_struct(tmp_path):
    """The binding's struct is the header's."""
    names = [n for n, _ in ec.PagedCache._fields_]
    src = tmp_path / "s.c"
    src.write_text('#include <stddef.h>\n#include <stdio.h>\n#include "edgecore.h"\nint main(void) {\nprintf("%zu", sizeof(EcPagedCache));\n'
                   + "".join(f'printf(" %zu", offsetof(EcPagedCache, {n}));\n' for n in names) + "return 0; }\n")
    subprocess.run(["gcc", str(src), "-I", str(REPO / "include"), "-o", str(tmp_path / "s")], check=True)
    got = subprocess.run([str(tmp_path / "s")], capture_output=True, text=True, timeout=20).stdout.split()
    assert [int(x) for x in got] == [C.sizeof(ec.PagedCache)] + [getattr(ec.PagedCache, n).offset for n in names]


def test_device_array_checks(tmp_path):
    exe = tmp_path / "pages_check"
    src = REPO / "tests" / "c" / "pages_check.c"
    subprocess.run(["gcc", "-std=c11", "-O1", "-Wall", "-fsanitize=undefined", "-fno-sanitize-recover=all",
                    "-I", str(REPO / "edgecore_amd" / "csrc"), str(src), "-o", str(exe)], check=True)
    p = subprocess.run([str(exe)], capture_output=True, text=True, timeout=60)
    assert p.returncode == 0 and " 0 wrong" in p.stdout, p.stdout + p.stderr


def pages(type="int8", **k):
    z, s = np.zeros((5, 2, 16, 64), np.uint8 if type != "fp16" else np.uint16), np.zeros((5, 2, 16), np.uint16)
    a = dict(type=type, k=z, v=z, table=np.zeros((2, 2), int), k_scale=None if type == "fp16" else s, v_scale=None if type == "fp16" else s)
    a.update(k)
    return ec.Pages(**a)


@pytest.mark.parametrize("k", [dict(type="int4"), dict(k=np.zeros((5, 2, 16, 64), np.int8)), dict(v=np.zeros((5, 2, 16, 32), np.uint8)),
                               dict(k_scale=None), dict(v_scale=np.zeros((5, 2, 15), np.uint16)), dict(table=[0, 1]),
                               dict(k_scale=np.zeros((5, 2, 16), np.float16))])
def test_pages_of_other_sizes(k):
    with pytest.raises(ValueError):
        pages(**k)


X, L = np.zeros((6, 4 * 64), np.float32), np.zeros((6, 50), np.float32)
Z = np.zeros((2, 30, 128), np.uint16)


@pytest.mark.parametrize("call", [
    lambda: ec.paged_append_dev(pages(), X, 1, [0, 0], [0, 3, 6]),
    lambda: ec.paged_append_dev(pages(), np.zeros((6, 8 * 64)), 2, [0, 0], [0, 3, 6]),
    lambda: ec.paged_append_dev(pages(), np.zeros((6, 6 * 64)), 2, [0, 0], [0, 3]),
    lambda: ec.paged_append_dev(pages(), np.zeros((6, 6 * 64)), 2, [0, 0]),
    lambda: ec.paged_append_dev(pages(), np.zeros((6, 6 * 64)), 2, [0, 0, 0], [0, 3, 4, 6]),
    lambda: ec.paged_append_dev(pages(), np.zeros((6, 6 * 64)), 2, [0, 0], [0, 3, 6], q_gamma=np.ones(63)),
    lambda: ec.attention_paged_dev(pages(), X, 3, [0, 0], [0, 3, 6]),
    lambda: ec.attention_paged_dev(pages(), X, 4, [0, 0], [0, 3, 6], out=X[:5]),
    lambda: ec.attention_paged_dev(pages(), X, 4, [0, 0]),
    lambda: ec.attention_paged_dev(pages(), X, 4, [0], [0, 6]),
    lambda: ec.paged_read_dev(pages(), Z, Z, [0, 0], [1]),
    lambda: ec.paged_read_dev(pages(), Z, Z[:1], [0, 0], [1, 1]),
    lambda: ec.paged_read_dev(pages(), Z, Z, [0, 0], [1, 1], slot=[0]),
    lambda: ec.paged_read_dev(pages(), Z[:, :, :64], Z[:, :, :64], [0, 0], [1, 1]),
    lambda: ec.logits_edit_dev(L, N=4),
    lambda: ec.logits_edit_dev(L, text=np.zeros((6, 3), int)),
    lambda: ec.logits_edit_dev(L, len=[0] * 6),
    lambda: ec.logits_edit_dev(L, text=np.zeros((5, 3), int), len=[0] * 6),
    lambda: ec.logits_edit_dev(L, bias=np.zeros((6, 3)), bias_token=np.zeros((6, 2), int)),
    lambda: ec.logits_edit_dev(L, mask=np.zeros((5, 2), np.uint32)),
    lambda: ec.logits_edit_dev(L, N=3, token=np.zeros((2, 2), int)),
    lambda: ec.logits_edit_dev(L, repetition=[1.0]),
    lambda: ec.logits_edit_dev(L, out=L[:5]),
])
def test_arrays_of_other_sizes(call):
    """The functions on host arrays refuse what the kernels would read past the end of."""
    with pytest.raises(ValueError):
        call()
