"""The operators that serve from a paged cache, as cases that can be timed.

A serving step over pages: the new rows' q and k are normalized, rotated and,
with v, written to the sequences' pages in 16 or 8 bits (ec_paged_append_dev),
the new tokens attend over them (ec_attention_paged_dev: one token or a chunk
for each sequence, with a window and first tokens that stay visible), a text's
rows come back as fp16 rows of the slot cache (ec_paged_read_dev), and logits
get their penalties, biases and masks (ec_logits_edit_dev).

`run` computes the plain forms in elementary torch operations, or with `own`
set calls the library (include/edgecore.h, bound by the edgecore_amd package).
The library runs on its own stream, so `prepare` waits for torch before it
returns.  Head shapes and vocabularies are those of the generator's presets:
GPT-2 small, Qwen2-0.5B and Qwen2.5-1.5B.
"""
import ctypes
import math

import numpy as np
import torch

own = False

V_GPT2, V_QWEN = 50257, 151936
HEADS = [(14, 2, 64), (12, 2, 128), (12, 12, 64)]  # H, KVH, head_dim of the presets
TYPES = ["fp16", "int8", "e4m3"]


# ---------------------------------------------------------------------------
# the cases
# ---------------------------------------------------------------------------

def listed():
    return [
        # one chat's next token: latency
        dict(name="attention_one", kind="attention", heads="14x2x64", type="fp16", page=16, B=1, n=1, rest=1, past=700,
             window=0, sinks=0),
        # 64 chats' next tokens over an int8 cache
        dict(name="attention_batch", kind="attention", heads="12x2x128", type="int8", page=16, B=64, n=1, rest=1,
             past=4000, window=0, sinks=0),
        # a chunk of a long prompt, after what the chunks before it left in the cache
        dict(name="attention_chunk", kind="attention", heads="14x2x64", type="e4m3", page=64, B=1, n=512, rest=1,
             past=7500, window=0, sinks=0),
        # a chunk of one sequence's prompt together with the next tokens of 23 others
        dict(name="attention_mixed", kind="attention", heads="14x2x64", type="int8", page=32, B=24, n=333, rest=1,
             past=1500, window=0, sinks=0),
        # chunks of multi-head sequences that see a window and their first tokens
        dict(name="attention_window", kind="attention", heads="12x12x64", type="int8", page=16, B=6, n=256, rest=256,
             past=5000, window=1000, sinks=4),
        # ragged prompts from their start: the largest
        dict(name="attention_prompt", kind="attention", heads="12x2x128", type="fp16", page=32, B=4, n=2048, rest=2048,
             past=0, window=0, sinks=0),
        # a token of 64 sequences into an int8 cache
        dict(name="append_batch", kind="append", heads="12x2x128", type="int8", page=16, B=64, n=1, rest=1, past=4000,
             norm=True, rot=128, layout=0),
        # ragged prompts into an e4m3 cache, interleaved pairs, no norm
        dict(name="append_prompt", kind="append", heads="14x2x64", type="e4m3", page=64, B=3, n=1000, rest=700, past=300,
             norm=False, rot=64, layout=1),
        # a chat's text into its slot
        dict(name="read_one", kind="read", heads="14x2x64", type="int8", page=16, B=1, past=1000),
        # long texts into theirs
        dict(name="read_batch", kind="read", heads="12x2x128", type="e4m3", page=64, B=8, past=16000),
        # one chat's logits with its penalties
        dict(name="edit_one", kind="edit", B=1, N=1, V=V_QWEN, text=1000, bias=0, mask=False),
        # the nodes of 8 trees, with biases and a grammar's mask
        dict(name="edit_tree", kind="edit", B=8, N=16, V=V_QWEN, text=4000, bias=32, mask=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["attention", "attention", "attention", "append", "read", "edit"])
    if kind == "edit":
        V = rng.choice([V_GPT2, V_QWEN, rng.randint(1000, 160000)])
        N = rng.choice([1, _log(rng, 2, 32)])
        return dict(kind=kind, B=_log(rng, 1, 128 // N), N=N, V=V, text=_log(rng, 1, 8000), bias=rng.choice([0, _log(rng, 1, 300)]),
                    mask=rng.random() < 0.5)
    H, KVH, hd = rng.choice(HEADS + [(16, 4, 96), (8, 1, 32), (10, 5, 80)])
    c = dict(kind=kind, heads="%dx%dx%d" % (H, KVH, hd), type=rng.choice(TYPES), page=rng.choice([16, 16, 32, 64, 128, 24]))
    if kind == "attention":
        while True:
            one = rng.random() < 0.4
            B = _log(rng, 1, 64)
            n = 1 if one else _log(rng, 2, 2048)
            c |= dict(B=B, n=n, rest=rng.choice([1, n]), past=rng.choice([0, _log(rng, 1, 30000), _log(rng, 1, 8000)]),
                      window=rng.choice([0, 0, _log(rng, 40, 4000)]))
            c["sinks"] = rng.choice([0, 4, 17]) if c["window"] else 0
            # what the plain form pads to and multiplies
            pairs = B * n * (c["past"] + n) * H
            if pairs <= 2.2e8 and work(c)["flops"] <= 5.0e10 and B * (c["past"] + n) * KVH * hd <= 7e7:
                return c
    if kind == "append":
        B = _log(rng, 1, 64)
        n = _log(rng, 1, max(2, 2048 // B))
        return c | dict(B=B, n=n, rest=rng.choice([1, n]), past=rng.choice([0, _log(rng, 1, 30000 // B)]),
                        norm=rng.random() < 0.6, rot=rng.choice([hd, hd, hd // 2 // 2 * 2]), layout=rng.choice([0, 0, 1]))
    B = _log(rng, 1, 8)
    return c | dict(B=B, past=_log(rng, 1, 120000 // B * 256 // max(256, KVH * hd)))


def _heads(c):
    return tuple(int(x) for x in c["heads"].split("x"))


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------

class PagedCache(ctypes.Structure):
    """include/edgecore.h, EcPagedCache"""
    _fields_ = [("k", ctypes.c_void_p), ("v", ctypes.c_void_p), ("k_scale", ctypes.c_void_p), ("v_scale", ctypes.c_void_p),
                ("type", ctypes.c_int), ("npages", ctypes.c_int), ("page", ctypes.c_int), ("KVH", ctypes.c_int),
                ("hd", ctypes.c_int), ("table", ctypes.c_void_p), ("ldt", ctypes.c_int)]


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed * 1000003 + 31)
    return g


def _normal(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _dev(a, dt):
    return torch.from_numpy(np.ascontiguousarray(a, dt)).cuda()


def _quantize(y, kind):
    """Rows [..., hd] as (codes, scales): one scale for a row, the nearest 16-bit
    value from below the largest over the codes' range on."""
    if kind == "fp16":
        return y.half(), None
    top = y.abs().amax(-1)
    t = top / (127.0 if kind == "int8" else 448.0)
    h = t.half()
    h = torch.where(h.float() < t, (h.view(torch.int16) + 1).view(torch.float16), h)
    z = y / torch.where(h > 0, h, torch.ones_like(h)).float()[..., None]
    if kind == "int8":
        return torch.round(z).clamp(-127, 127).to(torch.int8), h
    return z.clamp(-448, 448).to(torch.float8_e4m3fn), h


def _values(codes, scale):
    """What a row stands for: 16-bit values."""
    return codes if scale is None else (codes.float() * scale.float()[..., None]).half()


def _pages(c, r, g, s, rows, fill):
    """A cache whose pages lie in any order, and the sequences' tables: room for
    `rows` rows each."""
    _, KVH, hd = _heads(c)
    B, page = c["B"], c["page"]
    per = -(-rows // page)
    npages = B * per + 3
    shape = (npages, KVH, page, hd)
    names = ("k", "v")
    if c["type"] == "fp16":
        for n in names:
            s[n] = _normal(g, *shape).half() if fill else torch.zeros(shape, dtype=torch.float16, device="cuda")
            s[n + "s"] = None
    else:
        for n in names:
            # channels of unlike sizes, as keys have them
            y = _normal(g, *shape) * torch.exp(0.5 * _normal(g, hd)) if fill else torch.zeros(shape, device="cuda")
            s[n], s[n + "s"] = _quantize(y, c["type"])
    s["table"] = _dev(r.permutation(npages)[:B * per].reshape(B, per), np.int32)
    s["cache"] = PagedCache(s["k"].data_ptr(), s["v"].data_ptr(), *(None if s[n + "s"] is None else s[n + "s"].data_ptr() for n in names),
                            TYPES.index(c["type"]), npages, page, KVH, hd, s["table"].data_ptr(), per)


def _batch(c, r, s):
    """Lengths of cached text and of new rows that differ; the first sequence has
    all of both.  The call's rows behind the last sequence are padding."""
    B, n = c["B"], c["n"]
    past = r.integers(c["past"] - c["past"] // 4, c["past"] + 1, B)
    past[0] = c["past"]
    new = r.integers(max(1, c["rest"] - c["rest"] // 4), c["rest"] + 1, B)
    new[0] = n
    start = np.concatenate(([0], np.cumsum(new)))
    s.update(past=_dev(past, np.int32), start=_dev(start, np.int32), M=n + (B - 1) * c["rest"])


def _attention(c, seed, s):
    g, r = _gen(seed), np.random.default_rng(seed)
    H, KVH, hd = _heads(c)
    _batch(c, r, s)
    _pages(c, r, g, s, c["past"] + max(c["n"], c["rest"]), True)
    s.update(q=_normal(g, s["M"], H * hd), out=torch.zeros(s["M"], H * hd, device="cuda"))


def _append(c, seed, s):
    g, r = _gen(seed), np.random.default_rng(seed)
    H, KVH, hd = _heads(c)
    _batch(c, r, s)
    rows = c["past"] + max(c["n"], c["rest"])
    _pages(c, r, g, s, rows, False)
    n = c["rot"] // 2
    s.update(qkv=_normal(g, s["M"], (H + 2 * KVH) * hd) * 3.0, q=torch.zeros(s["M"], H * hd, device="cuda"),
             q_gamma=1.0 + 0.2 * _normal(g, hd) if c["norm"] else None,
             k_gamma=1.0 + 0.2 * _normal(g, hd) if c["norm"] else None,
             inv_freq=_dev(1e6 ** (-np.arange(n) / n), np.float64))
    # where the new rows are read back to: their sequence's slot
    most = max(c["n"], c["rest"])
    s.update(new=(s["start"][1:] - s["start"][:-1]).contiguous(), most=most,
             kc=torch.zeros(c["B"], most, KVH * hd, dtype=torch.float16, device="cuda"),
             vc=torch.zeros(c["B"], most, KVH * hd, dtype=torch.float16, device="cuda"))


def _read(c, seed, s):
    g, r = _gen(seed), np.random.default_rng(seed)
    _, KVH, hd = _heads(c)
    B, past = c["B"], c["past"]
    _pages(c, r, g, s, past, True)
    count = r.integers(past - past // 4, past + 1, B)
    count[0] = past
    s.update(first=_dev(np.zeros(B), np.int32), count=_dev(count, np.int32), slot=_dev(r.permutation(B), np.int32),
             kc=torch.zeros(B, past, KVH * hd, dtype=torch.float16, device="cuda"),
             vc=torch.zeros(B, past, KVH * hd, dtype=torch.float16, device="cuda"))


def _edit(c, seed, s):
    g, r = _gen(seed), np.random.default_rng(seed)
    B, N, V, T = c["B"], c["N"], c["V"], c["text"]
    x = _normal(g, B * N, V) * 2.0
    # texts repeat their likely tokens
    tokens = np.minimum((V * r.random((B, T)) ** 4).astype(np.int64), V - 1)
    length = r.integers(T - T // 4, T + 1, B)
    length[0] = T
    at = np.arange(N)
    s.update(logits=x, out=torch.zeros_like(x), text=_dev(tokens, np.int32), len=_dev(length, np.int32),
             prompt=_dev(length // 2, np.int32), repetition=_dev(r.uniform(1.0, 1.3, B), np.float32),
             frequency=_dev(r.uniform(0.0, 0.5, B), np.float32), presence=_dev(r.uniform(0.0, 0.5, B), np.float32),
             token=None, parent=None, nodes=None, bias_token=None, bias=None, nbias=None, mask=None)
    if N > 1:
        nodes = r.integers(max(1, N - N // 4), N + 1, B)
        nodes[B // 2] = N
        parent = np.where(at == 0, -1, np.maximum(at - r.integers(1, 5, (B, N)), 0))
        s.update(token=_dev(tokens[np.arange(B)[:, None], r.integers(0, T, (B, N))], np.int32), parent=_dev(parent, np.int32),
                 nodes=_dev(nodes, np.int32))
    if c["bias"]:
        k = min(c["bias"], V)
        s.update(bias_token=_dev(np.stack([r.choice(V, k, replace=False) for _ in range(B)]), np.int32),
                 bias=_dev(r.normal(0, 3, (B, k)), np.float32), nbias=_dev(r.integers(0, k + 1, B), np.int32))
    if c["mask"]:
        # a grammar's state allows a few tokens or most of them
        share = torch.from_numpy(r.choice([0.02, 0.5, 0.95], B * N).astype(np.float32)).cuda()[:, None]
        words = -(-V // 32)
        allow = torch.rand(B * N, words, 32, generator=g, device="cuda") < share[:, :, None]
        bits = (allow.long() << torch.arange(32, device="cuda")).sum(-1)
        s["mask"] = torch.where(bits >= 2 ** 31, bits - 2 ** 32, bits).int()


MAKE = {"attention": _attention, "append": _append, "read": _read, "edit": _edit}


def prepare(case, seed):
    s = dict(case=case)
    MAKE[case["kind"]](case, seed, s)
    torch.cuda.synchronize()
    return s


# ---------------------------------------------------------------------------
# one pass: the plain forms
# ---------------------------------------------------------------------------

def _place(s, rows):
    """The page and the row in it of each sequence's rows [B][n]."""
    page = s["case"]["page"]
    return s["table"].long().gather(1, (rows // page).clamp(0, s["table"].shape[1] - 1)), rows % page


def _rows(s, name, rows):
    """Rows [B][n] of the sequences' keys or values, [B][n][KVH][hd], in 16 bits."""
    p, o = _place(s, rows)
    scale = s[name + "s"]
    codes = s[name] if scale is None else s[name].view(torch.uint8)
    codes = codes[p, :, o]
    return _values(codes, None) if scale is None else _values(codes.view(s[name].dtype), scale[p, :, o])


def _plain_attention(s):
    c = s["case"]
    H, KVH, hd = _heads(c)
    B, G, N = c["B"], H // KVH, max(c["n"], c["rest"])
    L = c["past"] + N
    start, past = s["start"].long(), s["past"].long()
    at = torch.arange(N, device="cuda")
    live = at < (start[1:] - start[:-1])[:, None]
    row = torch.where(live, start[:-1, None] + at, 0)
    p = torch.arange(L, device="cuda")
    k = _rows(s, "k", p[None].expand(B, L)).float().permute(0, 2, 3, 1).contiguous()
    v = _rows(s, "v", p[None].expand(B, L)).float().transpose(1, 2).contiguous()
    q = s["q"][row].view(B, N, KVH, G, hd).permute(0, 2, 1, 3, 4).reshape(B, KVH, N * G, hd)
    t = (past[:, None] + at)[:, :, None]
    see = p <= t
    if c["window"]:
        see &= (p > t - c["window"]) | (p < c["sinks"])
    x = (q @ k).view(B, KVH, N, G, L) / math.sqrt(hd)
    x = x.masked_fill_(~see[:, None, :, None, :], -math.inf)
    x = torch.exp(x.sub_(x.amax(-1, keepdim=True)))
    x = x.div_(x.sum(-1, keepdim=True))
    o = (x.view(B, KVH, N * G, L) @ v).view(B, KVH, N, G, hd).permute(0, 2, 1, 3, 4).reshape(B, N, H * hd)
    out = s["out"]
    # rows of no sequence go to a row behind the last one
    full = torch.cat((out, out[:1]))
    full[torch.where(live, row, s["M"])] = o
    return full[:s["M"]]


def _plain_rotate(x, cos, sin, rot, layout):
    y, rest = x[..., :rot], x[..., rot:]
    if layout:
        a, b = y[..., 0::2], y[..., 1::2]
        y = torch.stack((a * cos - b * sin, a * sin + b * cos), -1).flatten(-2)
    else:
        a, b = y[..., :rot // 2], y[..., rot // 2:]
        y = torch.cat((a * cos - b * sin, a * sin + b * cos), -1)
    return torch.cat((y, rest), -1)


def _plain_append(s):
    c = s["case"]
    H, KVH, hd = _heads(c)
    M, B, most = s["M"], c["B"], s["most"]
    start, past = s["start"].long(), s["past"].long()
    x = s["qkv"].view(M, H + 2 * KVH, hd)
    q, k, v = x[:, :H], x[:, H:H + KVH], x[:, H + KVH:]
    if c["norm"]:
        q = q * torch.rsqrt(q.square().mean(-1, keepdim=True) + 1e-6) * s["q_gamma"]
        k = k * torch.rsqrt(k.square().mean(-1, keepdim=True) + 1e-6) * s["k_gamma"]
    m = torch.arange(M, device="cuda")
    seq = torch.bucketize(m, start[1:], right=True)
    live = seq < B
    seq = seq.clamp(max=B - 1)
    # positions times frequencies in 64 bits: far positions turn many times
    pos = past[seq] + m - start[seq]
    angle = pos.double()[:, None, None] * s["inv_freq"]
    cos, sin = torch.cos(angle).float(), torch.sin(angle).float()
    q = _plain_rotate(q, cos, sin, c["rot"], c["layout"])
    k = _plain_rotate(k, cos, sin, c["rot"], c["layout"])
    qo = torch.where(live[:, None], q.reshape(M, H * hd), s["q"])
    # into the pages: rows of no sequence to a page that no table names
    pg = s["table"].long()[seq, (pos // c["page"]).clamp(0, s["table"].shape[1] - 1)]
    used = torch.zeros(s["k"].shape[0], dtype=torch.bool, device="cuda").index_fill_(0, s["table"].long().view(-1), True)
    pg, off = torch.where(live, pg, used.int().argmin()), pos % c["page"]
    kq, ks = _quantize(k, c["type"])
    vq, vs = _quantize(v, c["type"])
    byte = torch.float16 if c["type"] == "fp16" else torch.uint8
    s["k"].view(byte)[pg, :, off] = kq.view(byte)
    s["v"].view(byte)[pg, :, off] = vq.view(byte)
    if ks is not None:
        s["ks"][pg, :, off] = ks
        s["vs"][pg, :, off] = vs
    # and back
    at = torch.arange(most, device="cuda")
    on = (at < s["new"][:, None])[:, :, None]
    rows = past[:, None] + torch.where(on[:, :, 0], at, 0)
    ko = torch.where(on, _rows(s, "k", rows).flatten(2), s["kc"])
    vo = torch.where(on, _rows(s, "v", rows).flatten(2), s["vc"])
    return qo, ko, vo


def _plain_read(s):
    c = s["case"]
    at = torch.arange(c["past"], device="cuda")
    on = (at < s["count"][:, None])[:, :, None]
    rows = s["first"].long()[:, None] + torch.where(on[:, :, 0], at, 0)
    slot = s["slot"].long()
    kc, vc = s["kc"], s["vc"]
    kc[slot] = torch.where(on, _rows(s, "k", rows).flatten(2), kc[slot])
    vc[slot] = torch.where(on, _rows(s, "v", rows).flatten(2), vc[slot])
    return kc, vc


def _ancestors(parent):
    """[B][N][N]: whether node j is i or one of its ancestors."""
    N = parent.shape[1]
    up = torch.nn.functional.one_hot(parent.long() + 1, N + 1)[:, :, 1:].float()
    a = up + torch.eye(N, device="cuda")
    a = (a @ a > 0).float()
    a = (a @ a > 0).float()
    a = (a @ a > 0).float()
    a = (a @ a > 0).float()
    a = (a @ a > 0).float()
    return a @ a > 0


def _plain_edit(s):
    c = s["case"]
    B, N, V = c["B"], c["N"], c["V"]
    x = s["logits"].view(B, N, V)
    at = torch.arange(c["text"], device="cuda")
    text = s["text"].long()
    inside = at < s["len"][:, None]
    said = inside & (at >= s["prompt"][:, None])
    zero = torch.zeros(B, V, device="cuda")
    every = zero.scatter_add(1, text, inside.float())[:, None]
    count = zero.scatter_add(1, text, said.float())[:, None]
    if s["token"] is not None:
        line = _ancestors(s["parent"]).float()
        node = torch.zeros(B, N, V, device="cuda").scatter_add_(2, s["token"].long()[:, None].expand(B, N, N), line)
        every, count = every + node, count + node
    r, f, p = (s[n][:, None, None] for n in ("repetition", "frequency", "presence"))
    y = torch.where(every > 0, torch.where(x > 0, x / r, x * r), x)
    y = y - f * count - torch.where(count > 0, p, 0.0)
    if s["bias"] is not None:
        on = torch.arange(s["bias"].shape[1], device="cuda") < s["nbias"][:, None]
        y = y + zero.scatter_add(1, s["bias_token"].long(), torch.where(on, s["bias"], 0.0))[:, None]
    if s["mask"] is not None:
        bit = s["mask"].view(B, N, -1)[:, :, :, None] >> torch.arange(32, dtype=torch.int32, device="cuda")
        y = y.masked_fill((bit.view(B, N, -1)[:, :, :V] & 1) == 0, -math.inf)
    if s["nodes"] is not None:
        y = torch.where((torch.arange(N, device="cuda") < s["nodes"][:, None])[:, :, None], y, s["out"].view(B, N, V))
    return y.view(B * N, V)


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------

def _p(t):
    return None if t is None else t.data_ptr()


def _ok(rc, what):
    if rc != 0:
        import edgecore_amd as ec
        raise RuntimeError("%s: %s" % (what, ec.last_error()))


def run(s):
    c, kind = s["case"], s["case"]["kind"]
    if not own:
        if kind == "attention":
            return {"out": _plain_attention(s)}
        if kind == "append":
            q, k, v = _plain_append(s)
            return {"q": q, "k": k, "v": v}
        if kind == "read":
            k, v = _plain_read(s)
            return {"k": k, "v": v}
        return {"out": _plain_edit(s)}
    import edgecore_amd as ec
    L = ec.lib()
    if kind == "edit":
        V = c["V"]
        _ok(L.ec_logits_edit_dev(_p(s["logits"]), V, _p(s["out"]), V, V, _p(s["text"]), c["text"], _p(s["len"]), _p(s["prompt"]),
                                 _p(s["token"]), _p(s["nodes"]), _p(s["parent"]), c["B"], c["N"], _p(s["repetition"]),
                                 _p(s["frequency"]), _p(s["presence"]), _p(s["bias_token"]), _p(s["bias"]), _p(s["nbias"]),
                                 0 if s["bias"] is None else s["bias"].shape[1], _p(s["mask"]), -(-V // 32)), "ec_logits_edit_dev")
        return {"out": s["out"]}
    H, KVH, hd = _heads(c)
    cache = ctypes.byref(s["cache"])
    if kind == "attention":
        _ok(L.ec_attention_paged_dev(cache, _p(s["q"]), H * hd, H, _p(s["start"]), _p(s["past"]), c["B"], s["M"], c["past"],
                                     c["window"], c["sinks"], _p(s["out"]), H * hd), "ec_attention_paged_dev")
        return {"out": s["out"]}
    if kind == "append":
        _ok(L.ec_paged_append_dev(cache, _p(s["qkv"]), (H + 2 * KVH) * hd, _p(s["q"]), H * hd, H, _p(s["q_gamma"]), _p(s["k_gamma"]),
                                  1e-6, _p(s["inv_freq"]), c["rot"], c["layout"], 1.0, _p(s["start"]), _p(s["past"]), c["B"],
                                  s["M"]), "ec_paged_append_dev")
        _ok(L.ec_paged_read_dev(cache, _p(s["past"]), _p(s["new"]), c["B"], s["most"], _p(s["kc"]), _p(s["vc"]), c["B"],
                                s["most"], None, None), "ec_paged_read_dev")
        return {"q": s["q"], "k": s["kc"], "v": s["vc"]}
    _ok(L.ec_paged_read_dev(cache, _p(s["first"]), _p(s["count"]), c["B"], c["past"], _p(s["kc"]), _p(s["vc"]), c["B"], c["past"],
                            _p(s["slot"]), None), "ec_paged_read_dev")
    return {"k": s["kc"], "v": s["vc"]}


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------

def work(case):
    c = case
    if c["kind"] == "edit":
        rows = c["B"] * (c["N"] - c["N"] // 8)
        return {"bytes": rows * c["V"] * 8 + (rows * c["V"] // 8 if c["mask"] else 0) + 4 * c["B"] * c["text"],
                "flops": 4.0 * rows * c["V"]}
    H, KVH, hd = _heads(c)
    row = 2 * KVH * (2 * hd if c["type"] == "fp16" else hd + 2)  # bytes of a cached row
    if c["kind"] == "read":
        rows = c["B"] * (c["past"] - c["past"] // 8)
        return {"bytes": rows * (row + 4 * KVH * hd), "flops": 2.0 * rows * KVH * hd}
    B, n, rest, past = c["B"], c["n"], c["rest"], c["past"] - c["past"] // 8  # the mean of the lengths
    rest -= rest // 8
    rows = n + (B - 1) * rest
    if c["kind"] == "append":
        return {"bytes": rows * (4 * hd * (2 * H + 2 * KVH) + 2 * row + 4 * KVH * hd), "flops": 12.0 * rows * (H + 2 * KVH) * hd}

    def pairs(n, past):  # (token, position) that n tokens see
        w = c["window"]
        if not w:
            return n * (past + (n + 1) / 2)
        return n * (min(w, past + (n + 1) / 2) + (c["sinks"] if past > w else 0))

    seen = pairs(n, c["past"]) + (B - 1) * pairs(rest, past)

    def span(n, past):
        return min(past + n, (c["window"] + n + c["sinks"]) if c["window"] else past + n)

    return {"bytes": 8 * rows * H * hd + row * (span(n, c["past"]) + (B - 1) * span(rest, past)), "flops": 4.0 * seen * H * hd}


# ---------------------------------------------------------------------------
# the same in 64 bits
# ---------------------------------------------------------------------------

def _exact_cache(s, name, b, n):
    """The first n rows of a sequence, [n][KVH][hd], in 64 bits: the 16-bit values
    that its codes and scales stand for."""
    page = s["case"]["page"]
    p = s["table"][b, :-(-n // page)].long()
    codes = s[name].view(torch.uint8)[p].view(s[name].dtype).double()
    if s[name + "s"] is not None:
        codes = (codes * s[name + "s"][p].double()[..., None]).half().double()
    return codes.permute(0, 2, 1, 3).flatten(0, 1)[:n]


def _exact_attention(c, s):
    H, KVH, hd = _heads(c)
    G = H // KVH
    out = s["out"].double()
    start, past = s["start"].tolist(), s["past"].tolist()
    for b in range(c["B"]):
        n = start[b + 1] - start[b]
        k, v = (_exact_cache(s, m, b, past[b] + n) for m in ("k", "v"))
        t = torch.arange(past[b], past[b] + n, device="cuda")[:, None]
        p = torch.arange(past[b] + n, device="cuda")
        hide = p > t
        if c["window"]:
            hide |= (p <= t - c["window"]) & (p >= c["sinks"])
        for h in range(H):
            q = s["q"][start[b]:start[b + 1], h * hd:(h + 1) * hd].double()
            x = (q @ k[:, h // G].t().contiguous()) * hd ** -0.5
            out[start[b]:start[b + 1], h * hd:(h + 1) * hd] = torch.softmax(x.masked_fill_(hide, -math.inf), 1) @ v[:, h // G].contiguous()
    return {"out": out}


def _exact_store(y, kind):
    """What a row of the cache stands for, from rows in 64 bits."""
    y = y.cpu().numpy()
    if kind == "fp16":
        return torch.from_numpy(y.astype(np.float16)).double()
    Q = 127.0 if kind == "int8" else 448.0
    t = np.abs(y).max(-1, keepdims=True) / Q
    h = t.astype(np.float16)
    h = np.where(h.astype(np.float64) < t, np.nextafter(h, np.float16(np.inf)), h)
    z = y / np.where(h > 0, h, 1).astype(np.float64)
    if kind == "int8":
        z = np.rint(z)
    else:  # e4m3: 3 bits behind the leading one, steps of 2^-9 below 2^-6
        e = np.maximum(np.floor(np.log2(np.maximum(np.abs(z), 2.0 ** -20))), -6)
        z = np.rint(z / 2.0 ** (e - 3)) * 2.0 ** (e - 3)
    return torch.from_numpy((np.clip(z, -Q, Q) * h.astype(np.float64)).astype(np.float16)).double()


def _exact_append(c, s):
    H, KVH, hd = _heads(c)
    rot = c["rot"]
    start, past = s["start"].tolist(), s["past"].tolist()
    q, kc, vc = s["q"].double(), s["kc"].double().cpu(), s["vc"].double().cpu()
    # element d of a head turns with its partner: d -> (partner, sign, frequency)
    d = np.arange(rot)
    partner = d ^ 1 if c["layout"] else (d + rot // 2) % rot
    which = torch.from_numpy(d // 2 if c["layout"] else d % (rot // 2)).cuda()
    sign = torch.from_numpy(np.where(partner > d, -1.0, 1.0)).cuda()
    partner = torch.from_numpy(partner).cuda()
    for b in range(c["B"]):
        n = start[b + 1] - start[b]
        pos = torch.arange(n, device="cuda").double() + past[b]
        angle = torch.outer(pos, s["inv_freq"])[:, which][:, None, :]
        x = s["qkv"][start[b]:start[b + 1]].view(n, H + 2 * KVH, hd).double()
        y = []
        for part, gamma in ((x[:, :H], s["q_gamma"]), (x[:, H:H + KVH], s["k_gamma"])):
            if gamma is not None:
                part = part / torch.sqrt((part * part).sum(-1, keepdim=True) / hd + 1e-6) * gamma.double()
            part = part.clone()
            turn = part[..., :rot]
            part[..., :rot] = turn * torch.cos(angle) + sign * turn[..., partner] * torch.sin(angle)
            y.append(part)
        q[start[b]:start[b + 1]] = y[0].reshape(n, -1)
        kc[b, :n] = _exact_store(y[1], c["type"]).reshape(n, -1)
        vc[b, :n] = _exact_store(x[:, H + KVH:], c["type"]).reshape(n, -1)
    return {"q": q, "k": kc, "v": vc}


def _exact_read(c, s):
    out = {}
    for name in ("k", "v"):
        to = s[name + "c"].double()
        for b, (n, slot) in enumerate(zip(s["count"].tolist(), s["slot"].tolist())):
            to[slot, :n] = _exact_cache(s, name, b, n).reshape(n, -1)
        out[name] = to
    return out


def _exact_edit(c, s):
    B, N, V = c["B"], c["N"], c["V"]
    x = s["logits"].cpu().numpy().astype(np.float64).reshape(B, N, V)
    y = s["out"].cpu().numpy().astype(np.float64).reshape(B, N, V)
    h = {n: None if s[n] is None else s[n].cpu().numpy() for n in ("text", "len", "prompt", "repetition", "frequency", "presence", "token",
                                                                   "parent", "nodes", "bias_token", "bias", "nbias", "mask")}
    for b in range(B):
        text = h["text"][b, :h["len"][b]]
        lines = []
        for i in range(N if h["nodes"] is None else h["nodes"][b]):
            line = []
            if h["token"] is not None:
                line = (lines[h["parent"][b, i]] if h["parent"][b, i] >= 0 else []) + [h["token"][b, i]]
                lines.append(line)
            said = np.concatenate((text[h["prompt"][b]:], np.array(line, text.dtype)))
            z = x[b, i].copy()
            seen = np.unique(np.concatenate((text, said)))
            r = float(h["repetition"][b])
            z[seen] = np.where(z[seen] > 0, z[seen] / r, z[seen] * r)
            t, n = np.unique(said, return_counts=True)
            z[t] -= float(h["frequency"][b]) * n + float(h["presence"][b])
            if h["bias"] is not None:
                k = h["nbias"][b]
                z[h["bias_token"][b, :k]] += h["bias"][b, :k]
            if h["mask"] is not None:
                z[np.unpackbits(h["mask"][b * N + i].view(np.uint8), bitorder="little")[:V] == 0] = -math.inf
            y[b, i] = z
    return {"out": torch.from_numpy(y.reshape(B * N, V))}


def exact(case, seed):
    s = prepare(case, seed)
    return {"attention": _exact_attention, "append": _exact_append, "read": _exact_read, "edit": _exact_edit}[case["kind"]](case, s)
