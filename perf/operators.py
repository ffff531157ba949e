"""The operators that verify drafted tokens, as cases that can be timed.

A serving step over the fp16 slot cache with a tree of drafted tokens for each
sequence (a chain of one token is an ordinary decode step): the new rows' q and
k are normalized, rotated and appended to the cache (ec_qk_norm_rope_dev), the
tree's nodes attend over the cache and their own ancestors
(ec_attention_tree_dev), every node's logits give a token (ec_sample_dev), and
the rows of the nodes that the tokens follow stay in the cache
(ec_tree_accept_dev).

`run` computes the plain forms in elementary torch operations, or with `own`
set calls the library (include/edgecore.h, bound by the edgecore_amd package).
The library runs on its own stream, so `prepare` waits for torch before it
returns.  Head shapes, widths and vocabularies are those of the generator's
presets: GPT-2 small, Qwen2-0.5B and Qwen2.5-1.5B.
"""
import math

import numpy as np
import torch

own = False

V_GPT2, V_QWEN = 50257, 151936
HEADS = [(14, 2, 64), (12, 2, 128), (12, 12, 64)]  # H, KVH, head_dim of the presets


# ---------------------------------------------------------------------------
# the cases
# ---------------------------------------------------------------------------

def listed():
    return [
        # one chat's next token, top-k and top-p as such servers set them: latency
        dict(name="sample_one", kind="sample", rows=1, V=V_QWEN, mode="topk"),
        # 16 sequences that sample from the nucleus of the whole vocabulary
        dict(name="sample_nucleus", kind="sample", rows=16, V=V_QWEN, mode="nucleus"),
        # every node of 8 trees of 16, each row with settings of its own
        # (greedy rows, min-p, no limit at all): the largest
        dict(name="sample_tree", kind="sample", rows=128, V=V_QWEN, mode="mixed"),
        # a draft of 8 tokens in one sequence of a chat's length
        dict(name="attention_one", kind="attention", heads="14x2x64", B=1, N=8, past=700, window=0, tree=True),
        # 16 ordinary decode steps, multi-head (GPT-2 small's context)
        dict(name="attention_decode", kind="attention", heads="12x12x64", B=16, N=1, past=1000, window=0, tree=False),
        # trees of 16 nodes in 8 sequences, grouped heads of 128
        dict(name="attention_batch", kind="attention", heads="12x2x128", B=8, N=16, past=4000, window=0, tree=True),
        # a wide tree over two contexts near the longest (32768): the largest
        dict(name="attention_long", kind="attention", heads="14x2x64", B=2, N=64, past=32600, window=0, tree=True),
        # the rows of 8 trees of 16 nodes
        dict(name="rope_tree", kind="rope", heads="14x2x64", B=8, N=16, past=4000, norm=True, rot=64, layout=0,
             scaling="yarn", tree=True),
        # three ragged prompts, interleaved pairs, part of a head of 80, no norm
        dict(name="rope_ragged", kind="rope", heads="10x5x80", B=3, N=333, past=0, norm=False, rot=32, layout=1,
             scaling="linear", tree=False),
        # a 2048-token prompt
        dict(name="rope_prompt", kind="rope", heads="12x2x128", B=1, N=2048, past=0, norm=True, rot=128, layout=0,
             scaling="none", tree=False),
        # one sequence's 8 nodes, 24 layers: latency
        dict(name="accept_one", kind="accept", kv=128, layers=24, B=1, N=8, past=700),
        # 16 sequences with wide trees, 28 layers
        dict(name="accept_batch", kind="accept", kv=256, layers=28, B=16, N=64, past=500),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["sample", "attention", "attention", "rope", "accept"])
    if kind == "sample":
        V = rng.choice([V_GPT2, V_QWEN, rng.randint(1000, 160000)])
        return dict(kind=kind, rows=_log(rng, 1, 120), V=V, mode=rng.choice(["plain", "topk", "nucleus", "minp", "mixed"]))
    if kind == "attention":
        while True:
            H, KVH, hd = rng.choice(HEADS + [(16, 4, 96), (8, 1, 32)])
            c = dict(kind=kind, heads="%dx%dx%d" % (H, KVH, hd), B=_log(rng, 1, 16), N=_log(rng, 1, 64),
                     past=_log(rng, 1, 30000), window=rng.choice([0, 0, 0, _log(rng, 40, 4000)]), tree=rng.random() < 0.7)
            w = work(c)
            if w["flops"] <= 1.1e10 and c["B"] * (c["past"] + c["N"]) <= 66000:
                return c
    if kind == "rope":
        H, KVH, hd = rng.choice(HEADS + [(16, 4, 96), (10, 5, 80), (9, 3, 42)])
        tree = rng.random() < 0.4
        B = _log(rng, 1, 16)
        N = _log(rng, 1, 64) if tree else _log(rng, 1, max(2, 2048 // B))
        return dict(kind=kind, heads="%dx%dx%d" % (H, KVH, hd), B=B, N=N, past=rng.choice([0, _log(rng, 1, 30000 // B)]),
                    norm=rng.random() < 0.6, rot=rng.choice([hd, hd, hd // 2 // 2 * 2]), layout=rng.choice([0, 0, 1]),
                    scaling=rng.choice(["none", "linear", "yarn"]), tree=tree)
    return dict(kind=kind, kv=rng.choice([128, 256, 768, 84]), layers=rng.randint(2, 28), B=_log(rng, 1, 16),
                N=_log(rng, 2, 64), past=_log(rng, 1, 500))


def _heads(c):
    return tuple(int(x) for x in c["heads"].split("x"))


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------

def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed * 1000003 + 29)
    return g


def _normal(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _dev(a, dt):
    return torch.from_numpy(np.ascontiguousarray(a, dt)).cuda()


def _trees(r, B, N, tree):
    """Parents [B][N] (-1 at the root): chains, or trees whose nodes hang on one
    of the few nodes before them."""
    at = np.arange(N)
    if not tree:
        return np.tile(at - 1, (B, 1))
    back = r.integers(1, 5, (B, N))
    return np.where(at == 0, -1, np.maximum(at - back, 0))


def _batch(c, r, s):
    """Slots in another order than the sequences, lengths of cached text and of
    drafts that differ (the longest has all of both)."""
    B, N = c["B"], c["N"]
    past = r.integers(c["past"] - c["past"] // 4, c["past"] + 1, B)
    past[0] = c["past"]
    nodes = r.integers(max(1, N - N // 4), N + 1, B)
    nodes[B // 2] = N
    s.update(slot=_dev(r.permutation(B), np.int32), past=_dev(past, np.int32), nodes=_dev(nodes, np.int32),
             C=c["past"] + N)


def _sample(c, seed, s):
    g, r = _gen(seed), np.random.default_rng(seed)
    R, V = c["rows"], c["V"]
    # logits of a language-model head: a few units of spread and a few likely tokens
    x = _normal(g, R, V) * 2.0
    likely = torch.randint(0, V, (R, 24), generator=g, device="cuda")
    s["logits"] = x.scatter_add_(1, likely, 6.0 + 3.0 * _normal(g, R, 24))
    mode = c["mode"]
    pick = r.integers(0, 6, R) if mode == "mixed" else None
    temp = r.uniform(0.5, 1.3, R)
    top_k, top_p, min_p = np.zeros(R), np.ones(R), np.zeros(R)
    if mode == "topk":
        top_k, top_p = r.integers(20, 101, R), r.uniform(0.8, 1.0, R)
    elif mode == "nucleus":
        top_p = r.uniform(0.7, 0.98, R)
    elif mode == "minp":
        min_p = r.uniform(0.02, 0.2, R)
    elif mode == "mixed":
        temp = np.where(pick == 0, 0.0, temp)
        top_k = np.where(pick == 1, r.integers(1, 101, R), np.where(pick == 2, r.integers(200, 5000, R), 0))
        top_p = np.where((pick == 1) | (pick == 3), r.uniform(0.5, 1.0, R), 1.0)
        min_p = np.where((pick == 3) | (pick == 4), r.uniform(0.001, 0.1, R), 0.0)
    s.update(temp=_dev(temp, np.float32), top_k=_dev(top_k, np.int32), top_p=_dev(top_p, np.float32),
             min_p=_dev(min_p, np.float32), u=_dev(r.random(R), np.float64),
             token=torch.zeros(R, dtype=torch.int32, device="cuda"), prob=torch.zeros(R, device="cuda"))


def _attention(c, seed, s):
    g, r = _gen(seed), np.random.default_rng(seed)
    H, KVH, hd = _heads(c)
    _batch(c, r, s)
    M = c["B"] * c["N"]
    s.update(q=_normal(g, M, H * hd), kc=_normal(g, c["B"], s["C"], KVH * hd).half(),
             vc=_normal(g, c["B"], s["C"], KVH * hd).half(), out=torch.zeros(M, H * hd, device="cuda"),
             parent=_dev(_trees(r, c["B"], c["N"], c["tree"]), np.int32))


def _inv_freq(c):
    """Rotary frequencies of theta 1e6: as they are, all divided by 4, or YaRN's
    ramp between the two over an original 4096 positions."""
    n = c["rot"] // 2
    f = 1e6 ** (-np.arange(n) / n)
    if c["scaling"] == "linear":
        return f / 4.0
    if c["scaling"] == "yarn":
        edge = [c["rot"] * math.log(4096 / (turns * 2 * math.pi)) / (2 * math.log(1e6)) for turns in (32.0, 1.0)]
        lo, hi = max(math.floor(edge[0]), 0), min(math.ceil(edge[1]), c["rot"] - 1)
        ramp = np.clip((np.arange(n) - lo) / max(hi - lo, 1), 0, 1)
        return f / 4.0 * ramp + f * (1 - ramp)
    return f


def _rope(c, seed, s):
    g, r = _gen(seed), np.random.default_rng(seed)
    H, KVH, hd = _heads(c)
    _batch(c, r, s)
    M = c["B"] * c["N"]
    s.update(qkv=_normal(g, M, (H + 2 * KVH) * hd) * 3.0, q=torch.zeros(M, H * hd, device="cuda"),
             kc=torch.zeros(c["B"], s["C"], KVH * hd, dtype=torch.float16, device="cuda"),
             vc=torch.zeros(c["B"], s["C"], KVH * hd, dtype=torch.float16, device="cuda"),
             q_gamma=1.0 + 0.2 * _normal(g, hd) if c["norm"] else None,
             k_gamma=1.0 + 0.2 * _normal(g, hd) if c["norm"] else None, inv_freq=_dev(_inv_freq(c), np.float64),
             factor=0.1 * math.log(4.0) + 1.0 if c["scaling"] == "yarn" else 1.0,
             parent=_dev(_trees(r, c["B"], c["N"], True), np.int32) if c["tree"] else None)


def _accept(c, seed, s):
    g, r = _gen(seed), np.random.default_rng(seed)
    B, N = c["B"], c["N"]
    _batch(c, r, s)
    parent = _trees(r, B, N, True)
    token, sampled = r.integers(0, V_QWEN, (B, N)), r.integers(0, V_QWEN, (B, N))
    # most nodes' sampled token is the one that one of their children drafted
    agree = r.random((B, N)) < 0.8
    agree[:, 0] = False
    b, i = np.nonzero(agree)
    sampled[b, parent[b, i]] = token[b, i]
    shape = (c["layers"], B, s["C"], c["kv"])
    s.update(kc=_normal(g, *shape).half(), vc=_normal(g, *shape).half(), parent=_dev(parent, np.int32),
             token=_dev(token, np.int32), sampled=_dev(sampled, np.int32))
    for name, n in (("path", (B, N)), ("npath", B), ("next", B), ("new_past", B)):
        s[name] = torch.zeros(n, dtype=torch.int32, device="cuda")


MAKE = {"sample": _sample, "attention": _attention, "rope": _rope, "accept": _accept}


def prepare(case, seed):
    s = dict(case=case)
    MAKE[case["kind"]](case, seed, s)
    torch.cuda.synchronize()
    return s


# ---------------------------------------------------------------------------
# one pass: the plain forms
# ---------------------------------------------------------------------------

def _plain_sample(s):
    x = s["logits"]
    v, at = torch.sort(x, dim=1, descending=True, stable=True)
    greedy = s["temp"] <= 0
    T = torch.where(greedy, torch.ones_like(s["temp"]), s["temp"]).double()[:, None]
    # sums over a vocabulary whose borders a given number may come near: 64 bits
    w = torch.exp((v.double() - v[:, :1].double()) / T)
    rank = torch.arange(x.shape[1], device="cuda")
    k = s["top_k"][:, None]
    w = torch.where((k > 0) & (rank >= k), 0.0, w)
    run_sum = torch.cumsum(w, 1)
    keep = (run_sum - w < s["top_p"].double()[:, None] * run_sum[:, -1:]) & (w >= s["min_p"].double()[:, None])
    keep[:, 0] = True
    w = torch.where(keep, w, 0.0)
    run_sum = torch.cumsum(w, 1)
    total = run_sum[:, -1:]
    hit = run_sum > s["u"][:, None] * total
    last = torch.where(w > 0, rank, 0).amax(1)
    pos = torch.where(hit.any(1), hit.int().argmax(1), last)
    pos = torch.where(greedy, torch.zeros_like(pos), pos)[:, None]
    prob = torch.where(greedy, 1.0, (w.gather(1, pos) / total)[:, 0])
    return at.gather(1, pos)[:, 0].int(), prob.float()


def _ancestors(parent):
    """[B][N][N]: whether node j is i or one of its ancestors."""
    N = parent.shape[1]
    up = torch.nn.functional.one_hot(parent.long() + 1, N + 1)[:, :, 1:].float()
    a = up + torch.eye(N, device="cuda")
    for _ in range(6):  # chains of up to 64 nodes
        a = (a @ a > 0).float()
    return a > 0


def _plain_attention(s):
    c = s["case"]
    H, KVH, hd = _heads(c)
    B, N, G, L = c["B"], c["N"], H // KVH, s["C"]
    anc = _ancestors(s["parent"])
    past = s["past"].long()[:, None, None]
    at = torch.arange(L, device="cuda")[None, None, :]
    inside = anc.gather(2, (at - past).clamp(0, N - 1).expand(B, N, L)) & (at >= past) & (at < past + N)
    see = (at < past) | inside
    if c["window"]:
        depth = anc.sum(2)[:, :, None] - 1
        # a node's place in the text, and a cache row's: its own, or its node's
        row = torch.where(at < past, at, past + (anc.sum(2) - 1)[:, None, :].gather(2, (at - past).clamp(0, N - 1)))
        see &= row > past + depth - c["window"]
    slot = s["slot"].long()
    k = s["kc"][slot].float().view(B, L, KVH, hd).permute(0, 2, 3, 1)
    v = s["vc"][slot].float().view(B, L, KVH, hd).permute(0, 2, 1, 3)
    q = s["q"].view(B, N, KVH, G, hd).permute(0, 2, 1, 3, 4).reshape(B, KVH, N * G, hd)
    x = (q @ k).view(B, KVH, N, G, L) / math.sqrt(hd)
    x = x.masked_fill(~see[:, None, :, None, :], -math.inf)
    p = torch.exp(x - x.amax(-1, keepdim=True))
    p = p / p.sum(-1, keepdim=True)
    o = (p.view(B, KVH, N * G, L) @ v).view(B, KVH, N, G, hd).permute(0, 2, 1, 3, 4).reshape(B, N, H * hd)
    live = torch.arange(N, device="cuda")[None, :] < s["nodes"][:, None]
    return torch.where(live[:, :, None], o, s["out"].view(B, N, H * hd)).view(B * N, H * hd)


def _plain_rotate(x, cos, sin, rot, layout):
    y, rest = x[..., :rot], x[..., rot:]
    if layout:
        a, b = y[..., 0::2], y[..., 1::2]
        y = torch.stack((a * cos - b * sin, a * sin + b * cos), -1).flatten(-2)
    else:
        a, b = y[..., :rot // 2], y[..., rot // 2:]
        y = torch.cat((a * cos - b * sin, a * sin + b * cos), -1)
    return torch.cat((y, rest), -1)


def _plain_rope(s):
    c = s["case"]
    H, KVH, hd = _heads(c)
    B, N = c["B"], c["N"]
    x = s["qkv"].view(B, N, H + 2 * KVH, hd)
    q, k, v = x[:, :, :H], x[:, :, H:H + KVH], x[:, :, H + KVH:]
    if c["norm"]:
        q = q * torch.rsqrt(q.square().mean(-1, keepdim=True) + 1e-6) * s["q_gamma"]
        k = k * torch.rsqrt(k.square().mean(-1, keepdim=True) + 1e-6) * s["k_gamma"]
    at = torch.arange(N, device="cuda")
    depth = at[None, :].expand(B, N) if s["parent"] is None else _ancestors(s["parent"]).sum(2) - 1
    # positions times frequencies in 64 bits: far positions turn many times
    angle = (s["past"][:, None] + depth).double()[:, :, None, None] * s["inv_freq"]
    cos, sin = (torch.cos(angle) * s["factor"]).float(), (torch.sin(angle) * s["factor"]).float()
    q = _plain_rotate(q, cos, sin, c["rot"], c["layout"])
    k = _plain_rotate(k, cos, sin, c["rot"], c["layout"])
    live = at[None, :] < s["nodes"][:, None]
    qo = torch.where(live[:, :, None], q.reshape(B, N, H * hd), s["q"].view(B, N, H * hd))
    slot, row = s["slot"].long()[:, None], s["past"].long()[:, None] + at
    kc, vc = s["kc"], s["vc"]
    kc[slot, row] = torch.where(live[:, :, None], k.reshape(B, N, KVH * hd).half(), kc[slot, row])
    vc[slot, row] = torch.where(live[:, :, None], v.reshape(B, N, KVH * hd).half(), vc[slot, row])
    return qo.view(B * N, H * hd), kc, vc


def _plain_accept(s):
    c = s["case"]
    N = c["N"]
    at = torch.arange(N, device="cuda")
    parent = s["parent"].long()
    up = parent.clamp(min=0)
    fits = (s["token"] == s["sampled"].gather(1, up)) & (at > 0) & (at < s["nodes"][:, None])
    # of siblings that fit the first one is taken
    same = (parent[:, :, None] == parent[:, None, :]) & fits[:, None, :] & (at[None, None, :] < at[None, :, None])
    good = (fits & ~same.any(2)) | (at == 0)
    taken = (~_ancestors(parent) | good[:, None, :]).all(2)
    npath = taken.sum(1)
    first = torch.sort(torch.where(taken, at, at + N), 1).values
    on = at < npath[:, None]
    path = torch.where(on, first, -1)
    nxt = s["sampled"].gather(1, path.gather(1, npath[:, None] - 1))[:, 0]
    slot, past = s["slot"].long()[:, None], s["past"].long()[:, None]
    to = past + at
    src = torch.where(on, past + path, to)
    kc, vc = s["kc"], s["vc"]
    kc[:, slot, to] = kc[:, slot, src]
    vc[:, slot, to] = vc[:, slot, src]
    return path.int(), npath.int(), nxt.int(), (s["past"] + npath).int()


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
        if kind == "sample":
            token, prob = _plain_sample(s)
            return {"token": token, "prob": prob}
        if kind == "attention":
            return {"out": _plain_attention(s)}
        if kind == "rope":
            q, kc, vc = _plain_rope(s)
            return {"q": q, "kc": kc, "vc": vc}
        path, npath, nxt, new_past = _plain_accept(s)
        return {"path": path, "npath": npath, "next": nxt, "past": new_past, "kc": s["kc"], "vc": s["vc"]}
    import edgecore_amd as ec
    L = ec.lib()
    if kind == "sample":
        _ok(L.ec_sample_dev(_p(s["logits"]), c["rows"], c["V"], c["V"], _p(s["temp"]), _p(s["top_k"]), _p(s["top_p"]),
                            _p(s["min_p"]), _p(s["u"]), _p(s["token"]), _p(s["prob"])), "ec_sample_dev")
        return {"token": s["token"], "prob": s["prob"]}
    tree = (_p(s["slot"]), _p(s["past"]), _p(s["nodes"]), _p(s["parent"]))
    if kind == "attention":
        H, KVH, hd = _heads(c)
        _ok(L.ec_attention_tree_dev(_p(s["q"]), H * hd, _p(s["kc"]), _p(s["vc"]), c["B"], s["C"], H, KVH, hd, *tree,
                                    c["B"], c["N"], c["past"], c["window"], _p(s["out"]), H * hd), "ec_attention_tree_dev")
        return {"out": s["out"]}
    if kind == "rope":
        H, KVH, hd = _heads(c)
        _ok(L.ec_qk_norm_rope_dev(_p(s["qkv"]), (H + 2 * KVH) * hd, _p(s["q"]), H * hd, _p(s["kc"]), _p(s["vc"]), c["B"],
                                  s["C"], H, KVH, hd, _p(s["q_gamma"]), _p(s["k_gamma"]), 1e-6, _p(s["inv_freq"]),
                                  c["rot"], c["layout"], s["factor"], *tree, c["B"], c["N"]), "ec_qk_norm_rope_dev")
        return {"q": s["q"], "kc": s["kc"], "vc": s["vc"]}
    _ok(L.ec_tree_accept_dev(_p(s["kc"]), _p(s["vc"]), c["layers"], c["B"], s["C"], c["kv"], *tree, _p(s["token"]),
                             _p(s["sampled"]), c["B"], c["N"], _p(s["path"]), _p(s["npath"]), _p(s["next"]),
                             _p(s["new_past"])), "ec_tree_accept_dev")
    return {"path": s["path"], "npath": s["npath"], "next": s["next"], "past": s["new_past"], "kc": s["kc"], "vc": s["vc"]}


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------

def work(case):
    c = case
    if c["kind"] == "sample":
        return {"bytes": 4 * c["rows"] * c["V"] + 32 * c["rows"], "flops": 3.0 * c["rows"] * c["V"]}
    B, N, past = c["B"], c["N"], c["past"] - c["past"] // 8  # the mean of the lengths
    if c["kind"] == "attention":
        H, KVH, hd = _heads(c)
        span = min(past, c["window"] or past) + min(N, 4)
        rows = B * (N - N // 8)
        return {"bytes": 8 * rows * H * hd + 4 * B * (min(past, (c["window"] or past) + N) + N) * KVH * hd,
                "flops": 4.0 * rows * span * H * hd}
    if c["kind"] == "rope":
        H, KVH, hd = _heads(c)
        rows = B * (N - N // 8)
        return {"bytes": rows * hd * (4 * (H + 2 * KVH) + 4 * H + 4 * KVH), "flops": 8.0 * rows * (H + KVH) * hd}
    # every sequence keeps some nodes; a kept row that stays in place moves nothing
    return {"bytes": 8 * c["layers"] * B * min(N - 1, 4) * c["kv"] + 16 * B * N, "flops": 2.0 * B * N}


# ---------------------------------------------------------------------------
# the same in 64 bits
# ---------------------------------------------------------------------------

def _exact_sample(c, s):
    x, R = s["logits"].cpu().numpy().astype(np.float64), c["rows"]
    T, K, P, Q, U = (s[n].cpu().numpy() for n in ("temp", "top_k", "top_p", "min_p", "u"))
    token, prob = np.zeros(R, np.int32), np.ones(R)
    for r in range(R):
        if T[r] <= 0:
            token[r] = int(np.argmax(x[r]))
            continue
        w = np.exp((x[r] - x[r].max()) / float(T[r]))
        order = np.argsort(-x[r], kind="stable")
        if K[r] > 0:
            order = order[:K[r]]
        before = np.concatenate(([0.0], np.cumsum(w[order])))
        n = int(np.searchsorted(before[:-1], float(P[r]) * before[-1], side="left"))
        order = order[:max(n, 1)]
        order = order[:max(int((w[order] >= float(Q[r])).sum()), 1)]
        total = np.cumsum(w[order])
        j = min(int(np.searchsorted(total, U[r] * total[-1], side="right")), len(order) - 1)
        token[r], prob[r] = order[j], w[order[j]] / total[-1]
    return {"token": torch.from_numpy(token), "prob": torch.from_numpy(prob)}


def _lineage(parent):
    """Each node's ancestors and itself, as lists, from the root down."""
    up = []
    for i, p in enumerate(parent):
        up.append((up[p] if p >= 0 else []) + [i])
    return up


def _exact_attention(c, s):
    H, KVH, hd = _heads(c)
    N, G = c["N"], H // KVH
    out = s["out"].double().view(c["B"], N, H * hd)
    parent = s["parent"].cpu().numpy()
    slot, past, nodes = (s[n].tolist() for n in ("slot", "past", "nodes"))
    for b in range(c["B"]):
        lines = _lineage(parent[b])
        n = past[b] + nodes[b]
        see = torch.zeros(nodes[b], n, dtype=torch.bool)
        for i in range(nodes[b]):
            lo = max(0, past[b] + len(lines[i]) - c["window"]) if c["window"] else 0
            see[i, lo:past[b]] = True
            near = lines[i][-c["window"]:] if c["window"] else lines[i]
            see[i, [past[b] + j for j in near]] = True
        see = see.cuda()
        for h in range(KVH):
            k, v = (s[m][slot[b], :n, h * hd:(h + 1) * hd].double() for m in ("kc", "vc"))
            for g in range(G):
                col = slice((h * G + g) * hd, (h * G + g + 1) * hd)
                x = s["q"].view(c["B"], N, H * hd)[b, :nodes[b], col].double() @ k.t().contiguous() * hd ** -0.5
                out[b, :nodes[b], col] = torch.softmax(x.masked_fill(~see, -math.inf), 1) @ v
    return {"out": out.reshape(c["B"] * N, H * hd)}


def _exact_rope(c, s):
    H, KVH, hd = _heads(c)
    N, rot = c["N"], c["rot"]
    slot, past, nodes = (s[n].tolist() for n in ("slot", "past", "nodes"))
    q, kc, vc = s["q"].double().view(c["B"], N, H * hd), s["kc"].double(), s["vc"].double()
    # element d of a head turns with its partner: d -> (partner, sign, frequency)
    d = np.arange(rot)
    partner = d ^ 1 if c["layout"] else (d + rot // 2) % rot
    which = d // 2 if c["layout"] else d % (rot // 2)
    sign = torch.from_numpy(np.where(partner > d, -1.0, 1.0)).cuda()
    partner = torch.from_numpy(partner).cuda()
    for b in range(c["B"]):
        n = nodes[b]
        depth = [len(x) - 1 for x in _lineage(s["parent"][b].tolist())][:n] if c["tree"] else list(range(n))
        pos = torch.tensor(depth, device="cuda").double() + past[b]
        angle = torch.outer(pos, s["inv_freq"])[:, torch.from_numpy(which).cuda()][:, None, :]
        x = s["qkv"].view(c["B"], N, H + 2 * KVH, hd)[b, :n].double()
        y = []
        for part, gamma in ((x[:, :H], s["q_gamma"]), (x[:, H:H + KVH], s["k_gamma"])):
            if gamma is not None:
                part = part / torch.sqrt((part * part).sum(-1, keepdim=True) / hd + 1e-6) * gamma.double()
            part = part.clone()
            turn = part[..., :rot]
            part[..., :rot] = s["factor"] * (turn * torch.cos(angle) + sign * turn[..., partner] * torch.sin(angle))
            y.append(part.reshape(n, -1))
        q[b, :n] = y[0]
        kc[slot[b], past[b]:past[b] + n] = y[1]
        vc[slot[b], past[b]:past[b] + n] = x[:, H + KVH:].reshape(n, -1)
    return {"q": q.reshape(c["B"] * N, H * hd), "kc": kc, "vc": vc}


def _exact_accept(c, s):
    B, N = c["B"], c["N"]
    parent, token, sampled = (s[n].cpu().numpy() for n in ("parent", "token", "sampled"))
    slot, past, nodes = (s[n].tolist() for n in ("slot", "past", "nodes"))
    kc, vc = s["kc"].double(), s["vc"].double()
    path, npath, nxt = np.full((B, N), -1, np.int32), np.zeros(B, np.int32), np.zeros(B, np.int32)
    for b in range(B):
        line = [0]
        while True:
            cur = line[-1]
            kids = [i for i in range(1, nodes[b]) if parent[b, i] == cur and token[b, i] == sampled[b, cur]]
            if not kids:
                break
            line.append(kids[0])
        path[b, :len(line)], npath[b], nxt[b] = line, len(line), sampled[b, line[-1]]
        rows = [past[b] + i for i in line]
        for cache in (kc, vc):
            cache[:, slot[b], past[b]:past[b] + len(line)] = cache[:, slot[b], rows].clone()
    return {"path": torch.from_numpy(path), "npath": torch.from_numpy(npath), "next": torch.from_numpy(nxt),
            "past": torch.from_numpy(npath + np.array(past, np.int32)), "kc": kc, "vc": vc}


def exact(case, seed):
    s = prepare(case, seed)
    return {"sample": _exact_sample, "attention": _exact_attention, "rope": _exact_rope,
            "accept": _exact_accept}[case["kind"]](case, s)
