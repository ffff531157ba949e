"""The operators for drafted tokens without a GPU: what their entry points
refuse (arguments are checked before the device is opened), the checks that the
kernels make of device arrays (ec_tree.h, compiled for the host), and the rotary
frequencies."""
import math
import subprocess

import numpy as np
import pytest

import edgecore_amd as ec

REPO = ec.PKG_DIR.parent
P = 4096  # stands for a device pointer: refused calls do not look at it


def refused(rc, *words):
    assert rc == -1, (rc, ec.last_error())
    for w in words:
        assert w in ec.last_error(), ec.last_error()


def sample(**k):
    a = dict(logits=P, rows=2, vocab=100, ld=100, temp=None, top_k=None, top_p=None, min_p=None, u=1 << 16, token=1 << 17,
             prob=None)
    a.update(k)
    return ec.lib().ec_sample_dev(*a.values())


def rope(**k):
    a = dict(qkv=P, ldx=4 * 64, q=1 << 17, ldq=128, kc=P, vc=P, nslots=2, C=100, H=2, KVH=1, hd=64, qg=None, kg=None, eps=1e-6,
             inv_freq=P, rot=64, layout=0, factor=1.0, slot=None, past=P, nodes=None, parent=None, B=2, N=3)
    a.update(k)
    return ec.lib().ec_qk_norm_rope_dev(*a.values())


def attention(**k):
    a = dict(q=P, ldq=128, kc=P, vc=P, nslots=2, C=100, H=2, KVH=1, hd=64, slot=None, past=P, nodes=None, parent=None,
             B=2, N=3, max_past=50, window=0, out=1 << 17, ldo=128)
    a.update(k)
    return ec.lib().ec_attention_tree_dev(*a.values())


def accept(**k):
    a = dict(kc=P, vc=P, layers=2, nslots=2, C=100, kv=128, slot=None, past=P, nodes=None, parent=P, token=P + 64, sampled=P + 128,
             B=2, N=3, path=P + 1024, npath=P + 2048, next=P + 2100, new_past=P + 2200)
    a.update(k)
    return ec.lib().ec_tree_accept_dev(*a.values())


@pytest.mark.parametrize("k", [dict(rows=-1), dict(vocab=0), dict(vocab=(1 << 18) + 1, ld=1 << 19), dict(ld=99),
                               dict(rows=(1 << 22) + 1), dict(logits=None), dict(u=None), dict(token=None),
                               dict(token=P + 2 * 400 - 4), dict(u=1 << 20, token=(1 << 20) + 12),
                               dict(temp=1 << 20, token=1 << 20), dict(token=1 << 20, prob=(1 << 20) + 4)])
def test_sample_refuses(k):
    refused(sample(**k), "ec_sample_dev")


def test_sample_no_rows():
    assert sample(rows=0) == 0


BATCH = [dict(B=0), dict(N=0), dict(B=-1), dict(N=-1), dict(B=65536), dict(B=65535, N=65), dict(nslots=0), dict(C=0),
         dict(past=None)]


@pytest.mark.parametrize("k", BATCH + [dict(N=65, parent=P), dict(H=0), dict(KVH=0), dict(H=3, KVH=2), dict(hd=0),
                                       dict(hd=513, ldx=1 << 20, ldq=1 << 20), dict(ldx=255), dict(ldq=127), dict(rot=63),
                                       dict(rot=66), dict(rot=-2), dict(layout=2), dict(layout=-1), dict(eps=-1e-6),
                                       dict(eps=math.nan), dict(qkv=None), dict(q=None), dict(kc=None), dict(vc=None),
                                       dict(inv_freq=None), dict(C=(1 << 30) + 1), dict(q=P), dict(q=P + 256, ldq=256),
                                       dict(q=P + 4 * (5 * 256 + 255))])
def test_rope_refuses(k):
    refused(rope(**k), "ec_qk_norm_rope_dev")


@pytest.mark.parametrize("k", BATCH + [dict(N=65), dict(H=3, KVH=2), dict(hd=513, ldq=2000, ldo=2000), dict(ldq=127),
                                       dict(ldo=127), dict(window=-1), dict(max_past=-1), dict(max_past=101),
                                       dict(q=None), dict(kc=None), dict(vc=None), dict(out=None), dict(out=P, ldo=256),
                                       dict(out=P + 512)])
def test_attention_refuses(k):
    refused(attention(**k), "ec_attention_tree_dev")


@pytest.mark.parametrize("k", BATCH + [dict(N=65), dict(layers=0), dict(kv=0), dict(kc=None), dict(vc=None),
                                       dict(token=None), dict(sampled=None), dict(path=None), dict(npath=None),
                                       dict(next=None), dict(new_past=None), dict(new_past=P), dict(npath=P + 4),
                                       dict(slot=P + 2096), dict(nodes=P + 2204),
                                       dict(parent=P + 1040), dict(token=P + 2048), dict(sampled=P + 1024),
                                       dict(npath=P + 2104), dict(next=P + 1044)])
def test_accept_refuses(k):
    refused(accept(**k), "ec_tree_accept_dev")


APART = dict(kc=1 << 24, vc=1 << 26)  # caches of their own
CACHE = 2 * 2 * 100 * 64              # bytes of one of rope() or attention()


@pytest.mark.parametrize("k", [dict(vc=(1 << 24) + CACHE - 2), dict(vc=1 << 24), dict(q=(1 << 24) + CACHE - 4),
                               dict(qkv=(1 << 26) - 4 * (5 * 256 + 256) + 4, past=P + 4), dict(past=1 << 17),
                               dict(qg=(1 << 26) + CACHE - 4), dict(kg=(1 << 17) + 4), dict(inv_freq=(1 << 26) - 252),
                               dict(slot=1 << 24), dict(nodes=(1 << 26) + 8), dict(parent=(1 << 17) - 20),
                               dict(nslots=2 ** 31 - 1, C=1 << 30, q=1 << 40)])
def test_rope_refuses_overlaps(k):
    refused(rope(**{**APART, "past": P * 4, **k}), "ec_qk_norm_rope_dev", "overlaps another array")


@pytest.mark.parametrize("k", [dict(out=(1 << 24) + CACHE - 4), dict(out=(1 << 26) - 4 * (5 * 128 + 128) + 4), dict(past=1 << 17),
                               dict(slot=(1 << 17) + 4), dict(nodes=(1 << 17) + 1000), dict(parent=(1 << 17) - 20),
                               dict(nslots=2 ** 31 - 1, C=1 << 30, out=1 << 40)])
def test_attention_refuses_overlaps(k):
    refused(attention(**{**APART, "past": P * 4, **k}), "ec_attention_tree_dev", "overlaps another array")


@pytest.mark.parametrize("k", [dict(vc=(1 << 24) + 2 * 2 * 2 * 100 * 128 - 2), dict(vc=1 << 24), dict(path=(1 << 24) - 4 * 6 + 4),
                               dict(npath=1 << 26), dict(token=(1 << 26) + 8), dict(parent=(1 << 24) + 400), dict(past=1 << 24),
                               dict(layers=2 ** 31 - 1, nslots=2 ** 31 - 1, next=1 << 40)])
def test_accept_refuses_overlaps(k):
    refused(accept(**{**APART, **k}), "ec_tree_accept_dev", "overlaps another array")


def test_accept_refuses_wide_rows():
    refused(accept(**APART, kv=(1 << 28) + 1), "ec_tree_accept_dev", "rows of")


def test_accept_refuses_more_layers_than_a_grid_has():
    refused(accept(**APART, layers=(1 << 20) + 1, nslots=1, C=1, kv=1), "ec_tree_accept_dev", "layers")


CACHE3, ROWS = np.zeros((2, 10, 64), np.uint16), np.zeros((6, 128), np.float32)
GOOD = {
    "rope": dict(qkv=np.zeros((6, 256), np.float32), kc=CACHE3, vc=CACHE3, H=2, KVH=1, past=[0, 1], N=3),
    "attention": dict(q=ROWS, kc=CACHE3, vc=CACHE3, H=2, KVH=1, past=[0, 1], N=3),
    "sample": dict(logits=ROWS, u=np.zeros(6)),
    "accept": dict(kc=CACHE3[None], vc=CACHE3[None], past=[0, 1], token=np.zeros((2, 3), int), sampled=np.zeros((2, 3), int)),
}
TREE = [dict(past=[0]), dict(past=[0, 1, 2]), dict(slot=[0]), dict(nodes=[3, 3, 3]), dict(parent=[-1, 0, 1]),
        dict(parent=np.zeros((3, 2), int)), dict(vc=CACHE3[:1]), dict(kc=CACHE3.astype(np.float16))]


@pytest.mark.parametrize("fn,k", [(f, k) for f in ("rope", "attention", "accept") for k in TREE] + [
    ("rope", dict(qkv=np.zeros((6, 255)))), ("rope", dict(qkv=np.zeros((7, 256)))), ("rope", dict(q=ROWS[:5])),
    ("rope", dict(q_gamma=np.ones(63))), ("rope", dict(k_gamma=np.ones(1))), ("rope", dict(KVH=3)),
    ("attention", dict(q=ROWS[:5])), ("attention", dict(H=3)), ("attention", dict(KVH=2)), ("attention", dict(out=ROWS[:5])),
    ("sample", dict(u=np.zeros(5))), ("sample", dict(temp=np.ones(1))), ("sample", dict(top_k=[1, 2])),
    ("sample", dict(top_p=np.ones(7))), ("sample", dict(min_p=np.ones((6, 2)))),
    ("accept", dict(sampled=np.zeros((2, 2), int)))])
def test_arrays_of_other_sizes(fn, k):
    """The functions on host arrays refuse what the kernels would read past the end of."""
    call = {"rope": ec.qk_norm_rope_dev, "attention": ec.attention_tree_dev, "sample": ec.sample_dev, "accept": ec.tree_accept_dev}[fn]
    if fn == "accept":
        k = {n: a[None] if n in ("kc", "vc") else a for n, a in k.items()}
    with pytest.raises(ValueError):
        call(**{**GOOD[fn], **k})


def test_numbers_of_more_than_32_bits(monkeypatch):
    monkeypatch.setattr(ec.DeviceBuffer, "from_array", classmethod(lambda cls, a: None))
    with pytest.raises((ValueError, OverflowError)):
        ec._Call().put("past", np.array([2 ** 32 + 5]), np.int32)
    with pytest.raises(ValueError):
        ec._Call().put("past", np.array([0.5]), np.int32)


def test_device_array_checks(tmp_path):
    exe = tmp_path / "tree_check"
    src = REPO / "tests" / "c" / "tree_check.c"
    subprocess.run(["gcc", "-std=c11", "-O1", "-Wall", "-fsanitize=undefined", "-fno-sanitize-recover=all",
                    "-I", str(REPO / "edgecore_amd" / "csrc"), str(src), "-o", str(exe)], check=True)
    p = subprocess.run([str(exe)], capture_output=True, text=True, timeout=60)
    assert p.returncode == 0 and " 0 wrong" in p.stdout, p.stdout + p.stderr


def test_rope_inv_freq():
    i = np.arange(32)
    plain = 1e6 ** (-2.0 * i / 64)
    # pow and the two divisions: a few units in the last place of 2^-53, times the exponent's size
    assert np.allclose(ec.rope_inv_freq(64, 1e6), plain, rtol=1e-14, atol=0)
    assert np.array_equal(ec.rope_inv_freq(64, 1e6, 2, 8.0), ec.rope_inv_freq(64, 1e6) / 8.0)
    assert np.allclose(ec.rope_inv_freq(64, 1e4, 3, 4.0), (1e4 * 4.0 ** (64 / 62)) ** (-2.0 * i / 64), rtol=1e-14, atol=0)
    yarn = ec.rope_inv_freq(64, 1e6, 1, 4.0, 4096.0)
    lo = math.floor(64 * math.log(4096 / (32 * 2 * math.pi)) / (2 * math.log(1e6)))
    hi = math.ceil(64 * math.log(4096 / (2 * math.pi)) / (2 * math.log(1e6)))
    ramp = np.clip((i - lo) / (hi - lo), 0, 1)
    assert np.allclose(yarn, plain / 4 * ramp + plain * (1 - ramp), rtol=1e-13, atol=0)
    assert yarn[0] == plain[0] and np.isclose(yarn[-1], plain[-1] / 4, rtol=1e-13)


@pytest.mark.parametrize("k", [(4, 64, 1e6, 1.0, 0.0), (-1, 64, 1e6, 1.0, 0.0), (0, 63, 1e6, 1.0, 0.0), (0, 0, 1e6, 1.0, 0.0),
                               (0, 64, 0.0, 1.0, 0.0), (0, 64, math.nan, 1.0, 0.0), (2, 64, 1e6, 0.0, 0.0),
                               (1, 64, 1e6, 4.0, 0.0), (1, 64, 1.0, 4.0, 4096.0)])
def test_rope_inv_freq_refuses(k):
    out = np.zeros(64)
    refused(ec.lib().ec_rope_inv_freq(*k, out.ctypes.data), "ec_rope_inv_freq")
    assert not out.any()
