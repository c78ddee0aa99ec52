"""The operators of a drafted-token step, in their plain form and as the library's entry points.

A step of speculative decoding takes a tree of drafted tokens per sequence through the model at
once. Around the quantized products it needs three operators:

* ``rope``: the rotary positions of the query and key heads (a node's position is its sequence's
  length plus its depth), with the rotated keys and the values stored in the KV cache;
* ``tree``: attention of every node over its sequence's cache and over its own ancestors;
* ``sample``: one token per row of logits, by temperature, top-k, top-p and min-p from a given
  uniform number.

``listed`` and ``draw`` give cases, ``prepare`` the inputs, ``run`` one pass: in plain torch
operations, or through sdy_rope_dev, sdy_tree_attention_dev and sdy_sample_dev where ``own`` is
set. ``exact`` gives the same results from the definitions in 64 bits.
"""
import ctypes
import math

import numpy as np
import torch

own = False

DTYPE = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
TYPE_ID = {"f32": 0, "f16": 1, "bf16": 30}  # ggml ids, as everywhere in the library


# ------------------------------------------------------------------------------------- cases

def listed():
    return [
        # One decoded token in the engine's own type: the latency of a call.
        dict(name="rope_one_f32", op="rope", type="f32", n_seq=1, per_seq=1, heads=16, kv=2, dim=128, rot=128,
             layout="half", scaling="none", far=2048),
        # Eight sequences' trees of 25 nodes each, past the trained context (bands by wavelength).
        dict(name="rope_trees_bf16", op="rope", type="bf16", n_seq=8, per_seq=25, heads=32, kv=8, dim=128, rot=128,
             layout="half", scaling="wavelength", far=131072),
        # A long prompt's chunk: the largest call.
        dict(name="rope_prompt_bf16", op="rope", type="bf16", n_seq=1, per_seq=8192, heads=32, kv=4, dim=128,
             rot=128, layout="half", scaling="dimension", far=40960),
        # Part of the head, pairs side by side, odd counts.
        dict(name="rope_part_f16", op="rope", type="f16", n_seq=3, per_seq=347, heads=15, kv=5, dim=80, rot=32,
             layout="interleaved", scaling="linear", far=8192),
        # One decoded token over a short cache in the engine's own type: latency again.
        dict(name="tree_one_f32", op="tree", type="f32", n_seq=1, nodes=1, heads=16, kv=2, dim=128, past=701,
             ragged=False, holes=False),
        # A small tree of one sequence.
        dict(name="tree_small_bf16", op="tree", type="bf16", n_seq=1, nodes=13, heads=32, kv=4, dim=128, past=4095,
             ragged=False, holes=False),
        # A serving batch, every sequence of its own length.
        dict(name="tree_batch_bf16", op="tree", type="bf16", n_seq=16, nodes=24, heads=32, kv=4, dim=128, past=8192,
             ragged=True, holes=False),
        # Wide trees over long contexts: the largest call.
        dict(name="tree_long_bf16", op="tree", type="bf16", n_seq=2, nodes=64, heads=32, kv=4, dim=128, past=65537,
             ragged=False, holes=False),
        # 64-wide heads, an odd tree with padding nodes, lengths from zero.
        dict(name="tree_odd_f16", op="tree", type="f16", n_seq=5, nodes=31, heads=9, kv=3, dim=64, past=2000,
             ragged=True, holes=True),
        # The token of one user's step from the whole vocabulary.
        dict(name="sample_one_f32", op="sample", type="f32", rows=1, vocab=151936, mode="usual", banned=False),
        # A batch whose requests all ask for something else, greedy ones among them.
        dict(name="sample_mixed_f32", op="sample", type="f32", rows=64, vocab=151936, mode="mixed", banned=False),
        # A batch of trees' nodes, most of the vocabulary excluded by a grammar.
        dict(name="sample_banned_bf16", op="sample", type="bf16", rows=333, vocab=49152, mode="mixed", banned=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


HEADS = [(9, 3, 64), (16, 2, 128), (32, 4, 128), (32, 8, 128), (14, 2, 64), (16, 8, 128), (15, 5, 80), (8, 1, 96)]
TREE_WORK = 2 * 32 * 64 * 65600 * 128  # query elements x keys of the largest listed tree case


def draw(rng):
    op = rng.choice(["rope", "tree", "sample"])
    kind = rng.choice(["f32", "f16", "bf16"])
    heads, kv, dim = rng.choice(HEADS)
    if op == "rope":
        n_seq = _log(rng, 1, 32)
        per = _log(rng, 1, 8192)
        per = max(1, min(per, 8192 * 36 * 128 // ((heads + kv) * dim * n_seq * (2 if kind == "f32" else 1))))
        return dict(op=op, type=kind, n_seq=n_seq, per_seq=per, heads=heads, kv=kv, dim=dim,
                    rot=rng.choice([dim, dim, dim // 2, 32]), layout=rng.choice(["half", "interleaved"]),
                    scaling=rng.choice(["none", "linear", "wavelength", "dimension"]),
                    far=max(per + 1, _log(rng, 1000, 1000000)))
    if op == "tree":
        n_seq, nodes, past = _log(rng, 1, 32), _log(rng, 1, 64), _log(rng, 1, 65537)
        most = TREE_WORK // (4 if kind == "f32" else 1)
        past = max(1, min(past, most // (n_seq * heads * nodes * dim) - nodes))
        past = max(1, min(past, (1 << 29) // (n_seq * kv * dim)))  # a cache of at most 2 x 2 GB
        return dict(op=op, type=kind, n_seq=n_seq, nodes=nodes, heads=heads, kv=kv, dim=dim, past=past,
                    ragged=rng.random() < 0.7, holes=rng.random() < 0.3)
    vocab = _log(rng, 1000, 262144)
    rows = max(1, min(_log(rng, 1, 400), 64 * 151936 // vocab))
    return dict(op=op, type=kind, rows=rows, vocab=vocab, mode=rng.choice(["usual", "mixed", "mixed", "whole"]),
                banned=rng.random() < 0.3)


def work(case):
    size = 4 if case["type"] == "f32" else 2
    if case["op"] == "rope":
        tok = case["n_seq"] * case["per_seq"]
        return dict(bytes=tok * (2 * (case["heads"] + 2 * case["kv"]) * case["dim"] * size + 12),
                    flops=tok * (case["heads"] + case["kv"]) * case["rot"] * 3)
    if case["op"] == "tree":
        keys = sum(n + case["nodes"] for n in _lengths(case))
        rows = case["n_seq"] * case["nodes"] * case["heads"]
        return dict(bytes=(2 * keys * case["kv"] + 2 * rows) * case["dim"] * size + rows // case["heads"] * 4,
                    flops=4 * keys * case["nodes"] * case["heads"] * case["dim"])
    n = case["rows"] * case["vocab"]
    return dict(bytes=n * size + case["rows"] * 28, flops=4 * n)


def _lengths(case):
    """Cached tokens of every sequence: ragged ones spread evenly from none to the whole length."""
    n, past = case["n_seq"], case["past"]
    return [past * s // max(1, n - 1) if case["ragged"] and n > 1 else past for s in range(n)]


# ------------------------------------------------------------------------------------- inputs

def _frequencies(case):
    """Radians per position of every rotated pair, and the factor on cosine and sine."""
    n, theta, factor, trained = case["rot"] // 2, 1e6, 4.0, 8192
    f = theta ** (-torch.arange(n, dtype=torch.float64) / n)
    if case["scaling"] == "linear":
        return f / factor, 1.0
    if case["scaling"] == "wavelength":  # kept where the trained context holds over 4 waves, stretched below 1
        keep = ((trained * f / (2 * math.pi) - 1.0) / (4.0 - 1.0)).clamp(0, 1)
        return f * keep + f / factor * (1 - keep), 1.0
    if case["scaling"] == "dimension":  # a ramp over the pairs between 32 waves and 1
        at = [2 * n * math.log(trained / (waves * 2 * math.pi)) / (2 * math.log(theta)) for waves in (32.0, 1.0)]
        lo, hi = max(math.floor(at[0]), 0), min(math.ceil(at[1]), 2 * n - 1)
        keep = 1 - ((torch.arange(n, dtype=torch.float64) - lo) / max(hi - lo, 0.001)).clamp(0, 1)
        return f * keep + f / factor * (1 - keep), 0.1 * math.log(factor) + 1
    return f, 1.0


def prepare(case, seed):
    g = torch.Generator("cuda").manual_seed(seed)
    st = dict(case)
    dt = DTYPE[case["type"]]

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32).to(dt)

    if case["op"] == "rope":
        n_seq, per, heads, kv, dim = (case[k] for k in ("n_seq", "per_seq", "heads", "kv", "dim"))
        tok = n_seq * per
        freq, st["mscale"] = _frequencies(case)
        st["freq"] = freq.cuda()
        # q, k and v are parts of one projection's rows, as the product of the joined weights leaves them
        qkv = normal(tok, heads + 2 * kv, dim)
        st["q"], st["k"], st["v"] = qkv[:, :heads], qkv[:, heads:heads + kv], qkv[:, heads + kv:]
        first = torch.randint(0, case["far"] - per, (n_seq, 1), generator=g, device="cuda")
        ahead = torch.arange(per, device="cuda")
        st["pos"] = (first + ahead).reshape(-1).to(torch.int32)
        st["rows"] = per + 3
        st["slot"] = (torch.arange(n_seq, device="cuda")[:, None] * st["rows"] + 2 + ahead).reshape(-1)
        st["q_out"] = torch.empty(tok, heads, dim, dtype=dt, device="cuda")
        st["k_cache"] = torch.zeros(n_seq, kv, st["rows"], dim, dtype=dt, device="cuda")
        st["v_cache"] = torch.zeros_like(st["k_cache"])
    elif case["op"] == "tree":
        n_seq, nodes, heads, kv, dim = (case[k] for k in ("n_seq", "nodes", "heads", "kv", "dim"))
        past = _lengths(case)
        st["rows"] = max(past) + nodes
        # scores of a standard deviation of 1.5, so that some keys stand out of a long cache
        st["q"] = (normal(n_seq, nodes, heads, dim) * 1.5).to(dt)
        st["k_cache"] = normal(n_seq, kv, st["rows"], dim)
        st["v_cache"] = normal(n_seq, kv, st["rows"], dim)
        st["n_past"] = torch.tensor(past, dtype=torch.int32, device="cuda")
        # node 0 continues the sequence; every other node hangs on an earlier one, mostly a near one
        at = torch.arange(nodes, device="cuda")
        back = (torch.rand(n_seq, nodes, generator=g, device="cuda") ** 2 * at).floor().long()
        parent = at - 1 - back.minimum((at - 1).clamp(min=0))
        if case["holes"]:  # shorter trees fill their rows with padding nodes
            parent[1::2, nodes - nodes // 3:] = -2
        st["parent"] = parent.to(torch.int32).contiguous()
        st["scale"] = dim ** -0.5
        st["out"] = torch.empty(n_seq, nodes, heads, dim, dtype=dt, device="cuda")
    else:
        rows, vocab = case["rows"], case["vocab"]
        x = torch.randn(rows, vocab, generator=g, device="cuda") * 2.5
        likely = torch.randint(0, vocab, (rows, 24), generator=g, device="cuda")
        x.scatter_(1, likely, torch.rand(rows, 24, generator=g, device="cuda") * 9 + 7)
        if case["banned"]:
            x[torch.rand(rows, vocab, generator=g, device="cuda") < 0.9] = -math.inf
            x.scatter_(1, likely[:, :4], torch.rand(rows, 4, generator=g, device="cuda") * 9 + 7)
        st["logits"] = x.to(dt)
        st["u"] = torch.rand(rows, generator=g, device="cuda")
        r = torch.arange(rows, device="cuda")
        one = torch.ones(rows, device="cuda")
        if case["mode"] == "usual":
            t, k, p, m = 0.8 * one, 40 * one, 0.95 * one, 0.0 * one
        elif case["mode"] == "whole":
            t, k, p, m = one, 0 * one, one, 0.0 * one
        else:  # each filter alone, all together, none, and greedy
            t = torch.where(r % 8 == 6, 0.0, 0.5 + (r % 5) * 0.2)
            k = torch.where(r % 4 == 1, 50.0, torch.where(r % 8 == 3, 1000.0, 0.0))
            p = torch.where((r % 4 == 2) | (r % 8 == 3), 0.9, 1.0)
            m = torch.where((r % 8 == 0) | (r % 8 == 3), 0.05, 0.0)
        st["temperature"], st["top_p"], st["min_p"] = t.float(), p.float(), m.float()
        st["top_k"] = k.to(torch.int32)
        st["id"] = torch.empty(rows, dtype=torch.int32, device="cuda")
        st["prob"] = torch.empty(rows, dtype=torch.float32, device="cuda")
    if own:  # the argument block and the workspace that a program keeps between its calls
        _arguments(st)
    return st


def _arguments(st):
    from sardyne_b200 import capi
    L = capi.lib()
    p = torch.Tensor.data_ptr
    kind = TYPE_ID[st["type"]]
    if st["op"] == "rope":
        q, k, v, c = st["q"], st["k"], st["v"], st["k_cache"]
        a = capi.RopeArgs(
            type=kind, n_tok=q.shape[0], n_head=st["heads"], n_kv_head=st["kv"], head_dim=st["dim"], n_rot=st["rot"],
            interleaved=int(st["layout"] == "interleaved"), mscale=st["mscale"], freq=p(st["freq"]), pos=p(st["pos"]),
            q=p(q), q_tok=q.stride(0), q_head=q.stride(1), q_out=p(st["q_out"]), q_out_tok=st["q_out"].stride(0),
            q_out_head=st["q_out"].stride(1), k=p(k), k_tok=k.stride(0), k_head=k.stride(1), v=p(v),
            v_tok=v.stride(0), v_head=v.stride(1), k_cache=p(c), v_cache=p(st["v_cache"]), slot=p(st["slot"]),
            n_seq=c.shape[0], max_seq=c.shape[2], cache_seq=c.stride(0), cache_head=c.stride(1), cache_row=c.stride(2))
        st["call"] = L.sdy_rope_dev
    elif st["op"] == "tree":
        q, c, o = st["q"], st["k_cache"], st["out"]
        a = capi.TreeAttentionArgs(
            type=kind, n_seq=st["n_seq"], n_node=st["nodes"], n_head=st["heads"], n_kv_head=st["kv"],
            head_dim=st["dim"], max_seq=c.shape[2], scale=st["scale"], q=p(q), q_seq=q.stride(0), q_node=q.stride(1),
            q_head=q.stride(2), k_cache=p(c), v_cache=p(st["v_cache"]), cache_seq=c.stride(0),
            cache_head=c.stride(1), cache_row=c.stride(2), n_past=p(st["n_past"]), parent=p(st["parent"]), out=p(o),
            out_seq=o.stride(0), out_node=o.stride(1), out_head=o.stride(2))
        need = L.sdy_tree_attention_bytes(ctypes.byref(a))
        st["ws"] = torch.empty(max(need, 1), dtype=torch.uint8, device="cuda")
        a.ws, a.ws_bytes = p(st["ws"]), need
        st["call"] = L.sdy_tree_attention_dev
    else:
        x = st["logits"]
        a = capi.SampleArgs(
            type=kind, n_row=x.shape[0], n_vocab=x.shape[1], row_stride=x.stride(0), logits=p(x),
            temperature=p(st["temperature"]), top_k=p(st["top_k"]), top_p=p(st["top_p"]), min_p=p(st["min_p"]),
            u=p(st["u"]), id=p(st["id"]), prob=p(st["prob"]))
        st["call"] = L.sdy_sample_dev
    st["args"], st["arg"] = a, ctypes.byref(a)


# ------------------------------------------------------------------------------------- one pass

def run(st):
    if own:
        if st["call"](st["arg"], torch.cuda.current_stream().cuda_stream) != 0:
            from sardyne_b200 import capi
            raise RuntimeError(capi.last_error())
        if st["op"] == "rope":
            return st["q_out"], st["k_cache"], st["v_cache"]
        return st["out"] if st["op"] == "tree" else (st["id"], st["prob"])
    return {"rope": _rope, "tree": _tree, "sample": _sample}[st["op"]](st)


def _rotated(x, cos, sin, rot, interleaved):
    y = x.float()
    r = y[..., :rot]
    a, b = (r[..., 0::2], r[..., 1::2]) if interleaved else (r[..., :rot // 2], r[..., rot // 2:])
    a, b = a * cos - b * sin, a * sin + b * cos
    r = torch.stack((a, b), -1).flatten(-2) if interleaved else torch.cat((a, b), -1)
    return torch.cat((r, y[..., rot:]), -1).to(x.dtype)


def _rope(st):
    angle = st["pos"].double()[:, None, None] * st["freq"]
    cos, sin = (torch.cos(angle) * st["mscale"]).float(), (torch.sin(angle) * st["mscale"]).float()
    inter = st["layout"] == "interleaved"
    st["q_out"].copy_(_rotated(st["q"], cos, sin, st["rot"], inter))
    seq, row = st["slot"] // st["rows"], st["slot"] % st["rows"]
    st["k_cache"][seq, :, row] = _rotated(st["k"], cos, sin, st["rot"], inter)
    st["v_cache"][seq, :, row] = st["v"]
    return st["q_out"], st["k_cache"], st["v_cache"]


def _tree(st):
    n_seq, nodes, heads, kv, dim = (st[k] for k in ("n_seq", "nodes", "heads", "kv", "dim"))
    rep, rows, dev = heads // kv, st["rows"], st["q"].device
    # which node stands on which: powers of the parent relation, and whether the path reaches a root
    parent = st["parent"].long()
    at = torch.arange(nodes, device=dev)
    step = (parent[:, :, None] == at) & (at < at[:, None])
    on = torch.linalg.matrix_power((step | (at == at[:, None])).double(), max(nodes, 2)) > 0
    on = on & (on & (parent == -1)[:, None, :]).any(-1, keepdim=True)
    key = torch.arange(rows, device=dev) - st["n_past"].long()[:, None]
    live = on.any(-1)
    sees = (key < 0)[:, None, :] & live[:, :, None]
    mine = on.gather(2, key.clamp(0, nodes - 1)[:, None, :].expand(n_seq, nodes, rows))
    sees = sees | (mine & ((key >= 0) & (key < nodes))[:, None, :])
    q = st["q"].float().view(n_seq, nodes, kv, rep, dim).permute(0, 2, 3, 1, 4).reshape(n_seq, kv, rep * nodes, dim)
    s = torch.matmul(q, st["k_cache"].float().transpose(-1, -2)) * st["scale"]
    s = s.view(n_seq, kv, rep, nodes, rows).masked_fill_(~sees[:, None, None], -math.inf)
    top = s.amax(-1, keepdim=True)
    s.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
    total = s.sum(-1, keepdim=True)
    o = torch.matmul(s.view(n_seq, kv, rep * nodes, rows), st["v_cache"].float()).view(n_seq, kv, rep, nodes, dim)
    o = torch.where(total > 0, o / total, 0.0)
    return o.permute(0, 3, 1, 2, 4).reshape(n_seq, nodes, heads, dim).to(st["q"].dtype)


def _sample(st):
    x = st["logits"].double()
    x = torch.where(torch.isnan(x), -math.inf, x)
    vocab = x.shape[1]
    t = st["temperature"].double()[:, None]
    greedy = ~(t > 0)
    top = x.amax(1, keepdim=True)
    w = torch.where(x == top, 0.0, (x - top) / torch.where(greedy, 1.0, t)).exp()
    order = torch.sort(x, dim=1, descending=True, stable=True).indices
    ws = w.gather(1, order)
    mass = ws.cumsum(1)
    k = st["top_k"].long()[:, None]
    k = torch.where(greedy, 1, torch.where(k <= 0, vocab, k.clamp(max=vocab)))
    p = st["top_p"].double()[:, None]
    np_ = (mass < p * mass.gather(1, k - 1)).sum(1, keepdim=True) + 1
    np_ = torch.where(p >= 1, vocab, np_)
    nm = (ws >= st["min_p"].double()[:, None].clamp(max=1)).sum(1, keepdim=True)
    n = torch.minimum(torch.minimum(k, np_), nm).clamp(min=1)
    place = torch.arange(vocab, device=x.device)
    kept = torch.zeros_like(w).scatter_(1, order, torch.where(place < n, ws, 0.0))
    c = kept.cumsum(1)
    total = c[:, -1:]
    last = torch.where(kept > 0, place, 0).amax(1, keepdim=True)
    i = torch.minimum((c <= st["u"].double()[:, None] * total).sum(1, keepdim=True), last)
    dead = top == -math.inf
    prob = torch.where(dead, 0.0, kept.gather(1, i) / total)
    return torch.where(dead, -1, i)[:, 0].to(torch.int32), prob[:, 0].float()


# ------------------------------------------------------------------------------------- 64 bits

def exact(case, seed):
    st = prepare(case, seed)
    return {"rope": _exact_rope, "tree": _exact_tree, "sample": _exact_sample}[case["op"]](st)


def _exact_rope(st):
    # every pair as a complex number, turned by the unit number of its angle
    unit = torch.polar(torch.full_like(st["freq"], st["mscale"])[None].expand(len(st["pos"]), -1).contiguous(),
                       st["pos"].double()[:, None] * st["freq"])[:, None]

    def turned(x):
        y = x.double().clone()
        n = st["rot"] // 2
        first, second = ((slice(0, 2 * n, 2), slice(1, 2 * n, 2)) if st["layout"] == "interleaved"
                         else (slice(0, n), slice(n, 2 * n)))
        z = torch.complex(y[..., first], y[..., second]) * unit
        y[..., first], y[..., second] = z.real, z.imag
        return y

    caches = []
    for x in (turned(st["k"]), st["v"].double()):
        c = st["k_cache"].double().permute(0, 2, 1, 3).reshape(-1, st["kv"], st["dim"]).clone()
        c[st["slot"]] = x
        caches.append(c.view(st["n_seq"], st["rows"], st["kv"], st["dim"]).permute(0, 2, 1, 3).contiguous())
    return turned(st["q"]), caches[0], caches[1]


def _exact_tree(st):
    out = torch.zeros(st["q"].shape, dtype=torch.float64, device="cuda")
    parents, lengths = st["parent"].tolist(), st["n_past"].tolist()
    rep = st["heads"] // st["kv"]
    for s, (par, past) in enumerate(zip(parents, lengths)):
        paths = []  # the nodes from each node to its root; none where the way ends elsewhere
        for i in range(st["nodes"]):
            path, j = [], i
            while j >= 0:
                path.append(j)
                j = par[j] if par[j] < j else -2
            paths.append(path if j == -1 else [])
        seen = torch.zeros(st["nodes"], past + st["nodes"], dtype=torch.bool)
        for i, path in enumerate(paths):
            if path:
                seen[i, :past] = True
                seen[i, [past + j for j in path]] = True
        live, seen = [i for i, path in enumerate(paths) if path], seen.cuda()
        if not live:
            continue
        for h in range(st["heads"]):
            k = st["k_cache"][s, h // rep, :past + st["nodes"]].double()
            v = st["v_cache"][s, h // rep, :past + st["nodes"]].double()
            score = (st["q"][s, live, h].double() @ k.T) * st["scale"]
            out[s, live, h] = torch.softmax(score.masked_fill(~seen[live], -math.inf), -1) @ v
    return out


def _exact_sample(st):
    x = st["logits"].float().cpu().numpy().astype(np.float64)
    t, p, m, u = (st[k].cpu().numpy().astype(np.float64) for k in ("temperature", "top_p", "min_p", "u"))
    ks = st["top_k"].cpu().numpy()
    ids, probs = np.full(len(x), -1, np.int32), np.zeros(len(x))
    for r, row in enumerate(x):
        finite = np.flatnonzero(row > -np.inf)
        if not finite.size:
            continue
        if not t[r] > 0:
            ids[r], probs[r] = finite[np.argmax(row[finite])], 1.0
            continue
        order = finite[np.argsort(-row[finite], kind="stable")]
        weight = np.exp((row[order] - row[order[0]]) / t[r])
        n = len(order) if ks[r] <= 0 else min(int(ks[r]), len(order))
        if p[r] < 1:
            n = min(n, 1 + int(np.searchsorted(np.cumsum(weight[:n]), p[r] * math.fsum(weight[:n]), "left")))
        n = max(1, min(n, int(np.count_nonzero(weight >= min(m[r], 1.0)))))
        by_index = np.argsort(order[:n])
        c = np.cumsum(weight[:n][by_index])
        at = min(int(np.searchsorted(c, u[r] * c[-1], "right")), n - 1)
        ids[r], probs[r] = order[:n][by_index[at]], weight[by_index[at]] / c[-1]
    return torch.from_numpy(ids), torch.from_numpy(probs)
