"""The drafted-token operators on the GPU against their definitions in 64 bits (drafted_ref.py)."""
import ctypes
import math

import numpy as np
import pytest

import drafted_ref as ref
from sardyne_b200 import capi

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

DTYPE = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
TYPE_ID = {"f32": 0, "f16": 1, "bf16": 30}
HALF = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}
KINDS = list(DTYPE)


@pytest.fixture(autouse=True)
def no_errors():
    capi.lib().sdy_clear_error()
    yield
    torch.cuda.synchronize()
    capi.check()


def f64(t):
    return t.detach().double().cpu().numpy()


def gen(seed):
    return torch.Generator("cuda").manual_seed(seed)


def randn(g, *shape, kind="f32"):
    return torch.randn(*shape, generator=g, device="cuda").to(DTYPE[kind])


def call(fn, args, stream=0):
    assert fn(ctypes.byref(args), stream) == 0, capi.last_error()


# ------------------------------------------------------------------------------------- rotary positions

def rope_args(kind, q, q_out, k, v, kc, vc, pos, freq, n_rot, interleaved, mscale=1.0, slot=None):
    p = torch.Tensor.data_ptr
    some = q if q is not None else k
    a = capi.RopeArgs(type=TYPE_ID[kind], n_tok=some.shape[0], n_head=0 if q is None else q.shape[1],
                      n_kv_head=0 if k is None else k.shape[1], head_dim=some.shape[2], n_rot=n_rot,
                      interleaved=interleaved, mscale=mscale, freq=p(freq) if n_rot else 0, pos=p(pos) if n_rot else 0)
    if q is not None:
        a.q, a.q_tok, a.q_head = p(q), q.stride(0), q.stride(1)
        a.q_out, a.q_out_tok, a.q_out_head = p(q_out), q_out.stride(0), q_out.stride(1)
    if k is not None:
        a.k, a.k_tok, a.k_head, a.k_cache = p(k), k.stride(0), k.stride(1), p(kc)
        a.n_seq, a.max_seq = kc.shape[0], kc.shape[2]
        a.cache_seq, a.cache_head, a.cache_row = kc.stride(0), kc.stride(1), kc.stride(2)
        if v is not None:
            a.v, a.v_tok, a.v_head, a.v_cache = p(v), v.stride(0), v.stride(1), p(vc)
        if slot is not None:
            a.slot = p(slot)
    return a


def close_rope(got, x, pos, freq, interleaved, mscale, kind):
    """cos and sin: the 32-bit functions err by at most 2 steps (2 x 2^-24 for values below 1), the
    reduced angle by 2^-27 pi < 2^-25, the factor by 2^-24: under 4 x 2^-24; the products and their
    sum add 2 more; the angle itself has 3 roundings of 2^-53. Then one rounding to the type."""
    want, size = ref.rope(f64(x), pos.cpu().numpy(), freq.cpu().numpy(), interleaved, mscale)
    angle = float(pos.abs().max()) * float(freq.max()) if len(freq) else 0.0
    tol = (6 * 2.0 ** -24 + 3 * angle * 2.0 ** -53) * size
    tol = tol + HALF[kind] * (abs(want) + tol) + 2.0 ** -25 * (kind == "f16")
    err = abs(f64(got) - want)
    assert (err <= tol).all(), (err - tol).max()
    n = 2 * len(freq)
    assert torch.equal(got[..., n:], x[..., n:])


ROPE = [  # tokens, heads, kv heads, head_dim, n_rot
    (1, 16, 2, 128, 128), (1, 1, 1, 2, 2), (7, 9, 3, 64, 64), (33, 15, 5, 80, 32), (5, 3, 1, 80, 40), (4, 4, 4, 33, 18),
    (3, 2, 1, 96, 96), (2, 5, 0, 128, 64), (6, 0, 2, 64, 32), (2, 1, 1, 1024, 1024), (3, 2, 2, 7, 0), (300, 8, 2, 64, 16)]


@pytest.mark.parametrize("interleaved", [0, 1])
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("shape", ROPE)
def test_rope(kind, shape, interleaved):
    tok, heads, kv, dim, rot = shape
    g = gen(tok * 1000 + dim + interleaved)
    qkv = randn(g, tok, heads + 2 * kv, dim, kind=kind)  # parts of one row, as a joined projection leaves them
    q, k, v = qkv[:, :heads], qkv[:, heads:heads + kv], qkv[:, heads + kv:]
    freq = torch.tensor(ref.rope_freqs(rot, 1e6) if rot else [], dtype=torch.float64, device="cuda")
    pos = torch.randint(0, 1 << 20, (tok,), generator=g, device="cuda", dtype=torch.int32)
    rows = tok + 5
    slot = torch.randperm(2 * rows, generator=g, device="cuda")[:tok]
    slot[tok // 2:tok // 2 + tok // 4] = torch.tensor(-1)  # padding tokens are not stored
    if tok > 2:
        slot[-1] = 2 * rows
    q_out = torch.full((tok, heads, dim), 7.0, device="cuda").to(DTYPE[kind])
    kc = torch.full((2, kv, rows, dim), 5.0, device="cuda").to(DTYPE[kind])
    vc = torch.full_like(kc, 3.0)
    a = rope_args(kind, q if heads else None, q_out, k if kv else None, v, kc, vc, pos, freq, rot, interleaved, 1.25, slot)
    call(capi.lib().sdy_rope_dev, a)
    if heads:
        close_rope(q_out, q, pos, freq, interleaved, float(np.float32(1.25)), kind)
    stored = [t for t in range(tok) if 0 <= int(slot[t]) < 2 * rows] if kv else []
    for c, x, fill in ((kc, k, 5.0), (vc, v, 3.0)):
        flat = c.permute(0, 2, 1, 3).reshape(2 * rows, kv, dim)
        at = slot[stored]
        if len(stored):
            if c is kc:
                close_rope(flat[at], x[stored], pos[stored], freq, interleaved, 1.25, kind)
            else:
                assert torch.equal(flat[at], x[stored])
        rest = torch.ones(2 * rows, dtype=torch.bool, device="cuda")
        rest[at] = False
        assert (flat[rest] == fill).all()


@pytest.mark.parametrize("kind,dim,rot,interleaved", [("bf16", 128, 128, 0), ("f32", 64, 32, 1), ("f16", 30, 30, 0)])
def test_rope_in_place_and_without_slots(kind, dim, rot, interleaved):
    g = gen(5)
    tok, heads = 17, 6
    buf = randn(g, tok, heads + 4, dim, kind=kind)
    before = buf.clone()
    q, k = buf[:, :heads], buf[:, heads:heads + 2]
    freq = torch.tensor(ref.rope_freqs(rot, 1e4), device="cuda")
    pos = torch.arange(-3, tok - 3, device="cuda", dtype=torch.int32)
    kc = torch.zeros(1, 2, tok, dim, device="cuda", dtype=DTYPE[kind])
    call(capi.lib().sdy_rope_dev, rope_args(kind, q, q, k, None, kc, None, pos, freq, rot, interleaved))
    close_rope(q, before[:, :heads], pos, freq, interleaved, 1.0, kind)
    close_rope(kc[0].transpose(0, 1), before[:, heads:heads + 2], pos, freq, interleaved, 1.0, kind)
    assert torch.equal(buf[:, heads:], before[:, heads:])


def test_rope_vector_and_scalar_forms_agree():
    """A buffer off the 16-byte boundary takes the element-wise kernel: the same values, bit for bit."""
    g = gen(6)
    tok, heads, dim = 9, 4, 64
    x = randn(g, tok, heads, dim, kind="bf16")
    freq = torch.tensor(ref.rope_freqs(dim, 1e6), device="cuda")
    pos = torch.randint(0, 1 << 17, (tok,), generator=g, device="cuda", dtype=torch.int32)
    outs = []
    for off in (0, 1):
        room = torch.zeros(x.numel() + 8, device="cuda", dtype=x.dtype)
        src = room[off:off + x.numel()].view_as(x)
        src.copy_(x)
        for inter in (0, 1):
            out = torch.empty_like(x)
            call(capi.lib().sdy_rope_dev, rope_args("bf16", src, out, None, None, None, None, pos, freq, dim, inter))
            outs.append(out)
    assert torch.equal(outs[0], outs[2]) and torch.equal(outs[1], outs[3])


def test_rope_far_positions():
    tok, dim = 6, 128
    x = randn(gen(8), tok, 2, dim)
    freq = torch.tensor(ref.rope_freqs(dim, 5e5), device="cuda")
    pos = torch.tensor([2 ** 31 - 1, -2 ** 31, 10 ** 9 + 7, 1 << 20, 131071, 0], device="cuda", dtype=torch.int32)
    out = torch.empty_like(x)
    call(capi.lib().sdy_rope_dev, rope_args("f32", x, out, None, None, None, None, pos, freq, dim, 0))
    close_rope(out, x, pos.long(), freq, 0, 1.0, "f32")
    assert torch.equal(out[5], x[5])


def test_rope_equals_the_engine_operator():
    """One token at a position the engine's own table holds: op_rope's rotation within its 32-bit
    steps (the table rounds cos and sin to 2^-25 each, as this kernel does within 4 x 2^-24)."""
    lib = capi.lib()
    heads, dim, at = 4, 64, 300
    x = randn(gen(9), 1, heads, dim)
    cos, sin = np.empty((at + 1, dim // 2), np.float32), np.empty((at + 1, dim // 2), np.float32)
    lib.op_rope_table(cos.ctypes.data, sin.ctypes.data, at + 1, dim, 1e4)
    freq = torch.tensor(ref.rope_freqs(dim, 1e4), device="cuda")
    pos = torch.tensor([at], device="cuda", dtype=torch.int32)
    for inter in (0, 1):
        host = x.cpu().numpy().copy()
        lib.op_rope(host.ctypes.data, heads, dim, cos[at].ctypes.data, sin[at].ctypes.data, inter)
        out = torch.empty_like(x)
        call(lib.sdy_rope_dev, rope_args("f32", x, out, None, None, None, None, pos, freq, dim, inter))
        _, size = ref.rope(f64(x), pos.cpu().numpy(), freq.cpu().numpy(), inter, 1.0)
        assert (abs(f64(out) - host) <= 9 * 2.0 ** -24 * size).all()


# ------------------------------------------------------------------------------------- tree attention

def random_parents(rng, n_seq, nodes, padding=True):
    parent = np.stack([np.array([rng.integers(-1, i) if rng.random() < 0.5 else i - 1 for i in range(nodes)])
                       for _ in range(n_seq)]).astype(np.int32)
    parent[:, 0] = -1
    if padding and nodes > 2:
        parent[-1, nodes // 2] = -2        # padding in the middle: its children are padding too
        parent[-1, nodes - 1] = nodes + 3  # not an earlier node
    return parent


def tree_args(kind, q, k, v, n_past, parent, out, scale, n_node=None, ws=None):
    p = torch.Tensor.data_ptr
    a = capi.TreeAttentionArgs(type=TYPE_ID[kind], n_seq=q.shape[0], n_node=q.shape[1], n_head=q.shape[2],
                               n_kv_head=k.shape[1], head_dim=q.shape[3], max_seq=k.shape[2], scale=scale, q=p(q),
                               q_seq=q.stride(0), q_node=q.stride(1), q_head=q.stride(2), k_cache=p(k), v_cache=p(v),
                               cache_seq=k.stride(0), cache_head=k.stride(1), cache_row=k.stride(2), n_past=p(n_past),
                               parent=0 if parent is None else p(parent), out=p(out), out_seq=out.stride(0),
                               out_node=out.stride(1), out_head=out.stride(2))
    need = capi.lib().sdy_tree_attention_bytes(ctypes.byref(a))
    assert need
    if ws is None:
        ws = torch.full((need,), 255, dtype=torch.uint8, device="cuda")  # NaN: nothing of it may be read unwritten
    a.ws, a.ws_bytes = p(ws), need
    a.keep = ws
    return a


def tree_case(kind, n_seq, nodes, heads, kv, dim, past, seed=0, parents=True, poison=True, room=9, q_scale=1.5):
    """Inputs with garbage (NaN, infinities) wherever no node may look: rows behind the drafted
    ones, rows of padding nodes."""
    rng = np.random.default_rng(seed + nodes + dim)
    g = gen(seed + nodes * 7 + dim)
    past = list(past)
    rows = max(past) + nodes + room
    q = randn(g, n_seq, nodes, heads, dim, kind=kind) * q_scale
    k, v = randn(g, n_seq, kv, rows, dim, kind=kind), randn(g, n_seq, kv, rows, dim, kind=kind)
    parent = random_parents(rng, n_seq, nodes) if parents else None
    clean = f64(k), f64(v)
    if poison:
        for s in range(n_seq):
            seen = ref.paths(parent[s] if parents else np.arange(nodes) - 1)
            dead = [past[s] + i for i in range(nodes) if not seen[i]] + list(range(past[s] + nodes, rows))
            k[s, :, dead] = float("nan")
            v[s, :, dead] = float("nan")
            v[s, :, dead[::2]] = float("inf")
            for i in dead:
                clean[0][s, :, i] = clean[1][s, :, i] = 0.0
    n_past = torch.tensor(past, dtype=torch.int32, device="cuda")
    return q, k, v, n_past, (torch.tensor(parent, device="cuda") if parents else None), parent, clean


def check_tree(kind, q, clean, n_past, parent, scale, out):
    want, tol = ref.tree_attention(f64(q), clean[0], clean[1], n_past.cpu().numpy(), parent, scale,
                                   0.0 if kind == "f32" else HALF[kind])
    got = f64(out)
    assert np.isfinite(got).all()
    if kind == "f32":
        tol = tol + HALF[kind] * abs(want)
    err = abs(got - want)
    assert (err <= tol).all(), ((err - tol).max(), np.argwhere(err > tol)[:4], err.max())
    for s in range(len(got)):
        for i, path in enumerate(ref.paths(parent[s] if parent is not None else np.arange(got.shape[1]) - 1)):
            if not path:
                assert not got[s, i].any()


TREES = [  # sequences, nodes, heads, kv heads, head_dim, cached tokens
    (1, 1, 1, 1, 8, [0]), (1, 1, 16, 2, 128, [0]), (1, 1, 16, 2, 128, [701]), (3, 1, 9, 3, 64, [0, 1, 130]),
    (2, 13, 8, 2, 128, [63, 64]), (2, 31, 9, 3, 64, [200, 0]), (1, 64, 8, 1, 128, [517]), (1, 33, 32, 4, 128, [127]),
    (4, 5, 14, 2, 64, [1000, 3, 65, 0]), (1, 17, 15, 5, 80, [95]), (2, 7, 8, 1, 96, [31, 129]), (1, 2, 4, 4, 256, [255]),
    (1, 100, 4, 2, 64, [40]), (1, 256, 2, 1, 64, [300]), (1, 3, 40, 1, 128, [77]), (2, 24, 4, 2, 40, [128, 257]),
    (1, 8, 2, 2, 200, [500])]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("shape", TREES)
def test_tree_attention(kind, shape):
    n_seq, nodes, heads, kv, dim, past = shape
    q, k, v, n_past, parent, par, clean = tree_case(kind, n_seq, nodes, heads, kv, dim, past)
    out = torch.full_like(q, float("nan"))
    a = tree_args(kind, q, k, v, n_past, parent, out, dim ** -0.5)
    call(capi.lib().sdy_tree_attention_dev, a)
    check_tree(kind, q, clean, n_past, par, dim ** -0.5, out)
    again = torch.full_like(q, float("nan"))
    call(capi.lib().sdy_tree_attention_dev, tree_args(kind, q, k, v, n_past, parent, again, dim ** -0.5))
    assert torch.equal(out, again)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("shape", [(2, 20, 4, 2, 256, [130, 7]), (1, 11, 8, 4, 136, [70]), (1, 70, 4, 2, 248, [65]),
                                   (40, 3, 14, 2, 72, [5 * i for i in range(40)]), (1, 9, 6, 3, 160, [3001])])
def test_tree_attention_rows_and_wide_heads(kind, shape):
    """One, two and several groups of rows of heads wider than the tensor cores' tiles; many sequences."""
    n_seq, nodes, heads, kv, dim, past = shape
    q, k, v, n_past, parent, par, clean = tree_case(kind, n_seq, nodes, heads, kv, dim, past, seed=5)
    out = torch.full_like(q, float("nan"))
    call(capi.lib().sdy_tree_attention_dev, tree_args(kind, q, k, v, n_past, parent, out, dim ** -0.5))
    check_tree(kind, q, clean, n_past, par, dim ** -0.5, out)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("nodes,heads,kv,past", [(1, 8, 2, 20011), (5, 4, 1, 9001), (24, 8, 2, 5003)])
def test_tree_attention_long(kind, nodes, heads, kv, past):
    """Long caches, which are split over the keys and joined."""
    q, k, v, n_past, parent, par, clean = tree_case(kind, 1, nodes, heads, kv, 64, [past], seed=3)
    out = torch.full_like(q, float("nan"))
    call(capi.lib().sdy_tree_attention_dev, tree_args(kind, q, k, v, n_past, parent, out, 0.125))
    check_tree(kind, q, clean, n_past, par, 0.125, out)


@pytest.mark.parametrize("kind", KINDS)
def test_tree_attention_chain(kind):
    """parent NULL: a causal chain."""
    q, k, v, n_past, _, _, clean = tree_case(kind, 2, 19, 4, 2, 64, [50, 0], parents=False)
    out = torch.full_like(q, float("nan"))
    call(capi.lib().sdy_tree_attention_dev, tree_args(kind, q, k, v, n_past, None, out, 0.125))
    check_tree(kind, q, clean, n_past, None, 0.125, out)


@pytest.mark.parametrize("kind", KINDS)
def test_tree_attention_rows_past_the_cache(kind):
    """Lengths beyond max_seq and below zero: rows that do not exist are not seen, nothing is read there."""
    rng = np.random.default_rng(2)
    g = gen(11)
    q = randn(g, 4, 6, 4, 64, kind=kind)
    k, v = randn(g, 4, 2, 70, 64, kind=kind), randn(g, 4, 2, 70, 64, kind=kind)
    n_past = torch.tensor([67, 70, 2 ** 31 - 1, -5], dtype=torch.int32, device="cuda")
    par = random_parents(rng, 4, 6, padding=False)
    out = torch.full_like(q, float("nan"))
    call(capi.lib().sdy_tree_attention_dev,
         tree_args(kind, q, k, v, n_past, torch.tensor(par, device="cuda"), out, 0.125))
    check_tree(kind, q, (f64(k), f64(v)), n_past, par, 0.125, out)


@pytest.mark.parametrize("kind", KINDS)
def test_tree_attention_only_padding(kind):
    """A whole tree of padding gives zeros, whatever the cache holds."""
    q = randn(gen(12), 2, 9, 4, 64, kind=kind)
    k = torch.full((2, 2, 80, 64), float("nan"), device="cuda", dtype=DTYPE[kind])
    parent = torch.full((2, 9), -2, dtype=torch.int32, device="cuda")
    n_past = torch.tensor([60, 0], dtype=torch.int32, device="cuda")
    out = torch.full_like(q, float("nan"))
    call(capi.lib().sdy_tree_attention_dev, tree_args(kind, q, k, k, n_past, parent, out, 0.125))
    assert not out.any()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_tree_attention_other_branch_is_not_seen(kind, bad):
    """A node that is not padding may hold NaN or infinities: the nodes off its path do not see them."""
    q, k, v, n_past, _, _, _ = tree_case(kind, 1, 12, 4, 2, 64, [70], parents=False, poison=False)
    par = np.array([[-1, 0, 0, 1, 2, 2, 3, -1, 7, 4, 8, 6]], np.int32)
    hurt = 2
    clean = f64(k), f64(v)
    k[0, :, 70 + hurt] = bad
    v[0, :, 70 + hurt, ::3] = bad
    out = torch.full_like(q, 9.0)
    call(capi.lib().sdy_tree_attention_dev,
         tree_args(kind, q, k, v, n_past, torch.tensor(par, device="cuda"), out, 0.125))
    free = [i for i, path in enumerate(ref.paths(par[0])) if hurt not in path]
    want, tol = ref.tree_attention(f64(q), *clean, n_past.cpu().numpy(), par, 0.125, HALF[kind])
    got = f64(out)
    assert len(free) == 8 and (abs(got - want)[:, free] <= tol[:, free]).all()


@pytest.mark.parametrize("kind", KINDS)
def test_tree_attention_strides(kind):
    """Queries out of a joined projection, a cache of [row][head] order, outputs into a wider buffer."""
    g = gen(13)
    n_seq, nodes, heads, kv, dim, rows = 2, 10, 6, 2, 64, 150
    joined = randn(g, n_seq, nodes, heads + 2 * kv, dim, kind=kind)
    q = joined[:, :, :heads]
    store = randn(g, 2, n_seq, rows, kv, dim, kind=kind)
    k, v = store[0].transpose(1, 2), store[1].transpose(1, 2)
    n_past = torch.tensor([rows - nodes, 17], dtype=torch.int32, device="cuda")
    par = random_parents(np.random.default_rng(4), n_seq, nodes)
    wide = torch.full((n_seq, nodes, heads + 3, dim), 4.0, device="cuda", dtype=DTYPE[kind])
    out = wide[:, :, 1:1 + heads]
    call(capi.lib().sdy_tree_attention_dev,
         tree_args(kind, q, k, v, n_past, torch.tensor(par, device="cuda"), out, 0.2))
    check_tree(kind, q, (f64(k), f64(v)), n_past, par, 0.2, out)
    assert (wide[:, :, 0] == 4).all() and (wide[:, :, 1 + heads:] == 4).all()


@pytest.mark.parametrize("kind", KINDS)
def test_tree_attention_large_scores(kind):
    """Scores that would overflow an exponential, falling and rising along the cache, and one key
    that takes all the weight late."""
    g = gen(14)
    q = torch.ones(1, 4, 4, 64, device="cuda", dtype=DTYPE[kind])
    for direction in (1, -1):
        ramp = torch.linspace(-4, 4, 400, device="cuda")[::1 if direction == 1 else 399].contiguous() if direction == 1 \
            else torch.linspace(4, -4, 400, device="cuda")
        k = ramp[None, None, :, None].expand(1, 2, 400, 64).contiguous().to(DTYPE[kind])
        v = randn(g, 1, 2, 400, 64, kind=kind)
        n_past = torch.tensor([396], dtype=torch.int32, device="cuda")
        out = torch.full_like(q, float("nan"))
        call(capi.lib().sdy_tree_attention_dev, tree_args(kind, q, k, v, n_past, None, out, 1.0))
        check_tree(kind, q, (f64(k), f64(v)), n_past, None, 1.0, out)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("scale", [0.0, -0.2, 1e-12])
def test_tree_attention_scales(kind, scale):
    """A scale of zero (all keys alike, masked ones none the less out), below zero, and tiny."""
    q, k, v, n_past, parent, par, clean = tree_case(kind, 2, 11, 4, 2, 64, [150, 5], seed=8)
    out = torch.full_like(q, float("nan"))
    call(capi.lib().sdy_tree_attention_dev, tree_args(kind, q, k, v, n_past, parent, out, scale))
    check_tree(kind, q, clean, n_past, par, float(np.float32(scale)), out)


@pytest.mark.parametrize("kind", KINDS)
def test_tree_attention_shared_cache(kind):
    """A sequence stride of zero: all sequences read one cache (it holds the same drafted rows too)."""
    g = gen(16)
    q = randn(g, 3, 5, 4, 64, kind=kind)
    k, v = (randn(g, 1, 2, 140, 64, kind=kind).expand(3, 2, 140, 64) for _ in range(2))
    n_past = torch.tensor([130, 7, 64], dtype=torch.int32, device="cuda")
    out = torch.full_like(q, float("nan"))
    call(capi.lib().sdy_tree_attention_dev, tree_args(kind, q, k, v, n_past, None, out, 0.125))
    check_tree(kind, q, (f64(k), f64(v)), n_past, None, 0.125, out)


def test_tree_attention_many_sequences():
    """More sequences than threads of a block, most of them short: every share holds several."""
    n_seq = 900
    past = [(37 * s) % 300 for s in range(n_seq)]
    for kind in ("bf16", "f32"):
        g = gen(17)
        q = randn(g, n_seq, 2, 2, 64, kind=kind)
        k, v = randn(g, n_seq, 1, 302, 64, kind=kind), randn(g, n_seq, 1, 302, 64, kind=kind)
        n_past = torch.tensor(past, dtype=torch.int32, device="cuda")
        out = torch.full_like(q, float("nan"))
        call(capi.lib().sdy_tree_attention_dev, tree_args(kind, q, k, v, n_past, None, out, 0.125))
        check_tree(kind, q, (f64(k), f64(v)), n_past, None, 0.125, out)


def test_tree_attention_far_offsets():
    """Elements past 2^32 of a cache in HBM: the last sequence's rows lie behind them."""
    n_seq, kv, dim = 3, 1, 64
    rows = 2 ** 31 // dim + 1000  # one sequence alone passes 2^31 elements
    store = torch.empty(n_seq * kv * rows * dim, device="cuda", dtype=torch.bfloat16)  # 13 GB
    k = store.view(n_seq, kv, rows, dim)
    g = gen(15)
    for s in range(n_seq):
        k[s, :, :300] = randn(g, kv, 300, dim, kind="bf16")
    q = randn(g, n_seq, 4, 2, dim, kind="bf16")
    n_past = torch.tensor([290, 200, 296], dtype=torch.int32, device="cuda")
    out = torch.full_like(q, float("nan"))
    call(capi.lib().sdy_tree_attention_dev, tree_args("bf16", q, k, k, n_past, None, out, 0.125))
    near = k[:, :, :300].contiguous()
    check_tree("bf16", q, (f64(near), f64(near)), n_past, None, 0.125, out)
    del store, k


# ------------------------------------------------------------------------------------- sampling

def sample(logits, u, kind="f32", temperature=None, top_k=None, top_p=None, min_p=None, prob=True, stream=0):
    rows, vocab = logits.shape
    p = torch.Tensor.data_ptr
    keep = dict(u=torch.as_tensor(u, dtype=torch.float32, device="cuda"))
    for name, value, dt in (("temperature", temperature, torch.float32), ("top_k", top_k, torch.int32),
                            ("top_p", top_p, torch.float32), ("min_p", min_p, torch.float32)):
        if value is not None:
            keep[name] = torch.as_tensor(value, device="cuda").to(dt).expand(rows).contiguous()
    ids = torch.full((rows + 1,), -77, dtype=torch.int32, device="cuda")
    probs = torch.full((rows + 1,), -77.0, device="cuda")
    a = capi.SampleArgs(type=TYPE_ID[kind], n_row=rows, n_vocab=vocab, row_stride=logits.stride(0), logits=p(logits),
                        id=p(ids), prob=p(probs) if prob else 0, **{n: p(t) for n, t in keep.items()})
    call(capi.lib().sdy_sample_dev, a, stream)
    torch.cuda.synchronize()
    assert ids[rows] == -77 and probs[rows] == -77
    return ids[:rows].cpu().numpy(), f64(probs[:rows])


def check_sample(logits, u, got, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """Choices are equal: the masses carry 2^-45 each, so a choice differs only where the uniform
    number lies within n 2^-45 of a border. prob: the mass's rounding, the sum's and one to 32 bits."""
    x, (ids, probs) = f64(logits), got
    rows, vocab = x.shape
    every = lambda v: np.broadcast_to(np.asarray(v, np.float64), (rows,))  # noqa: E731
    t, k, p, m, u = every(temperature), every(top_k), every(top_p), every(min_p), every(u)
    for r in range(rows):
        # the parameters as the kernel gets them
        want, prob = ref.sample(np.where(np.isnan(x[r]), -np.inf, x[r]), float(np.float32(u[r])),
                                float(np.float32(t[r])), int(k[r]), float(np.float32(p[r])), float(np.float32(m[r])))
        assert ids[r] == want, (r, ids[r], want, t[r], k[r], p[r], m[r])
        assert abs(probs[r] - prob) <= 2.0 ** -23 * prob + vocab * 2.0 ** -44


VOCABS = [1, 2, 31, 32, 33, 1000, 1025, 4097, 49152, 151936, 262147, 400000]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("vocab", VOCABS)
def test_sample_filters(kind, vocab):
    g = gen(vocab)
    rows = 12
    x = (randn(g, rows, vocab) * 3).to(DTYPE[kind])
    u = torch.rand(rows, generator=g, device="cuda").cpu().numpy()
    u[0], u[1] = 0.0, 1 - 2.0 ** -24
    r = np.arange(rows)
    settings = [dict(), dict(temperature=0.7), dict(top_k=40), dict(top_k=1), dict(top_p=0.9), dict(min_p=0.1),
                dict(top_k=3000, top_p=0.8), dict(temperature=1.5, top_k=50, top_p=0.95, min_p=0.05),
                dict(temperature=np.where(r % 3 == 0, 0.0, 0.5 + r / 8), top_k=np.where(r % 2, 0, 7 + 100 * r),
                     top_p=np.where(r % 4 == 1, 0.5, 1.0), min_p=np.where(r % 5 == 2, 0.02, 0.0))]
    for s in settings:
        check_sample(x, u, sample(x, u, kind, **s), **s)


@pytest.mark.parametrize("kind,rows,vocab", [("f32", 20, 1500), ("f16", 40, 1500), ("bf16", 160, 1500), ("f32", 160, 9001),
                                             ("bf16", 80, 60001), ("f32", 30, 70001)])
def test_sample_many_rows(kind, rows, vocab):
    """Rows enough that each has one CTA, two or four."""
    g = gen(rows + vocab)
    x = (randn(g, rows, vocab) * 3).to(DTYPE[kind])
    x[::3, ::2] = -float("inf")
    u = torch.rand(rows, generator=g, device="cuda").cpu().numpy()
    r = np.arange(rows)
    s = dict(temperature=np.where(r % 7 == 6, 0.0, 0.5 + r % 5 / 4), top_k=np.select([r % 6 == 1, r % 6 == 3, r % 6 == 4], [40, 900, 600]),
             top_p=np.where((r % 6 == 2) | (r % 6 == 3), 0.9, 1.0), min_p=np.where(r % 6 == 5, 0.05, 0.0))
    check_sample(x, u, sample(x, u, kind, **s), **s)
    check_sample(x[:, 1:], u, sample(x[:, 1:], u, kind, top_p=0.95), top_p=0.95)


@pytest.mark.parametrize("temperature", [1e-40, 1e-30, 1e-3, 1e20, 3e38])
@pytest.mark.parametrize("span", [1e-30, 1.0, 3e38])
def test_sample_ranges(temperature, span):
    """Temperatures and logits from one end of the type to the other."""
    g = gen(31)
    x = (torch.rand(3, 2000, generator=g, device="cuda") * 2 - 1) * span
    x[1] = x[1].abs()
    x[2, 100:] = x[2, 7]
    u = np.array([0.3, 0.6, 0.9], np.float32)
    for s in (dict(), dict(top_k=30), dict(top_k=700), dict(top_p=0.6), dict(min_p=0.7), dict(min_p=1.0)):
        check_sample(x, u, sample(x, u, temperature=temperature, **s), temperature=temperature, **s)


@pytest.mark.parametrize("kind", KINDS)
def test_sample_ties(kind):
    """Equal logits rank by index, in every filter; whole rows of one value too."""
    rows, vocab = 8, 20000
    g = gen(3)
    x = torch.randint(0, 4, (rows, vocab), generator=g, device="cuda").to(DTYPE[kind])
    x[1] = 2.5
    x[2, 100:] = -float("inf")
    u = torch.linspace(0, 0.999, rows).numpy()
    for s in (dict(), dict(top_k=40), dict(top_k=9000), dict(top_p=0.5), dict(top_p=0.25, top_k=64), dict(min_p=1.0),
              dict(min_p=0.2), dict(top_p=0.0), dict(temperature=0.0), dict(temperature=1e-30), dict(temperature=1e30)):
        check_sample(x, u, sample(x, u, kind, **s), **s)


@pytest.mark.parametrize("spread", [1e-2, 1e-5, 30.0])
def test_sample_narrow_and_wide(spread):
    """Logits so close that a bucket of distances holds thousands of different ones, and far apart."""
    g = gen(21)
    rows, vocab = 6, 50001
    x = randn(g, rows, vocab) * spread
    u = torch.rand(rows, generator=g, device="cuda").cpu().numpy()
    for s in (dict(), dict(top_k=7), dict(top_k=511), dict(top_k=512), dict(top_k=513), dict(top_k=20000), dict(top_p=0.3),
              dict(top_p=0.999), dict(top_k=30000, top_p=0.5, min_p=0.01), dict(temperature=0.01, top_p=0.9)):
        check_sample(x, u, sample(x, u, **s), **s)


def test_sample_zeros_of_both_signs():
    """-0 and 0 are the same logit: the lower index goes first."""
    x = torch.full((4, 64), -1.0, device="cuda")
    x[:, 9], x[:, 30], x[:, 31] = -0.0, 0.0, -0.0
    u = np.array([0.0, 0.3, 0.6, 0.9], np.float32)
    for s in (dict(top_k=1), dict(top_k=2), dict(top_k=3), dict(temperature=0.0), dict(top_p=0.1), dict(min_p=1.0)):
        got = sample(x, u, **s)
        check_sample(x + 0.0, u, got, **s)
    assert (sample(x, u, temperature=0.0)[0] == 9).all()


def test_sample_infinite_temperature():
    """All weights alike; an infinite logit still takes everything."""
    x = torch.linspace(-5, 5, 1000, device="cuda").repeat(3, 1)
    x[1, 17] = float("inf")
    x[2, ::2] = -float("inf")
    u = np.array([0.25, 0.5, 0.75], np.float32)
    for s in (dict(), dict(top_k=10), dict(top_p=0.5), dict(min_p=0.5)):
        check_sample(x, u, sample(x, u, temperature=float("inf"), **s), temperature=float("inf"), **s)


def test_sample_special_values():
    inf, nan = float("inf"), float("nan")
    x = torch.full((9, 300), -inf, device="cuda")
    x[0, 7] = 1.0                      # one live logit
    x[1, 5:9] = inf                    # infinities share the weight
    x[1, 20] = 3.0
    x[2] = nan                         # nothing to take
    x[4, ::2] = nan                    # NaN is never taken
    x[4, 1::2] = torch.linspace(-3, 3, 150)
    x[5] = -3e38
    x[5, 250] = 3e38
    x[6] = torch.finfo(torch.float32).min  # a mask of the type's lowest value, everywhere
    x[7] = torch.linspace(-80, 80, 300)
    x[8, 299] = -1e30
    u = np.full(9, 0.6, np.float32)
    for s in (dict(), dict(top_k=3), dict(top_p=0.7), dict(min_p=0.5), dict(temperature=0.0), dict(top_k=3, top_p=0.5, min_p=0.1)):
        got = sample(x, u, **s)
        check_sample(x, u, got, **s)
        assert got[0][2] == -1 and got[0][3] == -1 and got[1][3] == 0
    check_sample(x, u * 0, sample(x, u * 0 + np.float32(nan)))         # NaN counts as 0
    check_sample(x, u * 0, sample(x, u * 0 - 4))
    check_sample(x, u * 0 + 1 - 2.0 ** -24, sample(x, u * 0 + 1.5))    # clamped below 1
    off = dict(temperature=1.0, top_p=nan, min_p=nan, top_k=-3)
    check_sample(x, u, sample(x, u, **off))
    check_sample(x, u, sample(x, u, temperature=nan), temperature=0.0)
    check_sample(x, u, sample(x, u, temperature=-1.0), temperature=0.0)
    check_sample(x, u, sample(x, u, min_p=7.0), min_p=1.0)
    check_sample(x, u, sample(x, u, top_k=10 ** 9, top_p=2.0))


def test_sample_strides_and_no_prob():
    g = gen(4)
    buf = randn(g, 5, 1200)
    for first in (0, 1):  # a row start off the 16-byte boundary
        x = buf[:, first:first + 1001]
        u = np.linspace(0, 0.99, 5).astype(np.float32)
        got = sample(x, u, top_k=20)
        check_sample(x, u, got, top_k=20)
        assert np.array_equal(sample(x, u, top_k=20, prob=False)[0], got[0])
    one = buf[:1].expand(64, 1200)  # one row, many numbers
    u = (np.arange(64) / 64).astype(np.float32)
    check_sample(one, u, sample(one, u, top_p=0.8), top_p=0.8)


def test_sample_distribution():
    """65536 choices from one row: every token's count within 5 standard deviations of n p."""
    x = torch.tensor([[0.0, 1.0, 2.0, -1.0, 3.0, 2.0, -float("inf"), 0.5]], device="cuda").expand(65536, 8)
    u = np.random.default_rng(0).permutation(65536).astype(np.float32) / 65536
    ids, _ = sample(x, u, temperature=0.8)
    w = np.exp(f64(x[0]) / float(np.float32(0.8)))
    n = np.bincount(ids, minlength=8)
    # u runs over an even grid, so each count is n p to within its two ends
    assert (abs(n - 65536 * w / w.sum()) <= 2).all()


# ------------------------------------------------------------------------------------- together, streams, graphs

class Step:
    """One drafted-token step on one layer: rotary positions and the store, tree attention over the
    updated cache, logits by a product, one token per node."""

    def __init__(self, kind="bf16", seed=0, n_seq=2, nodes=12, heads=8, kv=2, dim=64, past=(90, 37), vocab=500):
        g = gen(seed)
        rng = np.random.default_rng(seed)
        self.kind, self.dim, self.nodes, self.heads, self.kv, self.past = kind, dim, nodes, heads, kv, list(past)
        tok = n_seq * nodes
        self.qkv = randn(g, tok, heads + 2 * kv, dim, kind=kind)
        rows = max(past) + nodes
        self.kc, self.vc = randn(g, n_seq, kv, rows, dim, kind=kind), randn(g, n_seq, kv, rows, dim, kind=kind)
        self.k0, self.v0 = self.kc.clone(), self.vc.clone()
        self.par = random_parents(rng, n_seq, nodes, padding=False)
        depth = np.array([[len(path) - 1 for path in ref.paths(p)] for p in self.par])
        self.pos = torch.tensor((np.array(past)[:, None] + depth).reshape(-1), dtype=torch.int32, device="cuda")
        self.slot = torch.tensor([s * rows + past[s] + i for s in range(n_seq) for i in range(nodes)], device="cuda")
        self.freq = torch.tensor(ref.rope_freqs(dim, 1e4), device="cuda")
        self.n_past = torch.tensor(past, dtype=torch.int32, device="cuda")
        self.parent = torch.tensor(self.par, device="cuda")
        self.q = torch.empty(n_seq, nodes, heads, dim, device="cuda", dtype=DTYPE[kind])
        self.att = torch.empty_like(self.q)
        self.w = randn(g, heads * dim, vocab) * (heads * dim) ** -0.5 * 4
        self.logits = torch.empty(tok, vocab, device="cuda")
        self.u = torch.rand(tok, generator=g, device="cuda")
        self.ids = torch.full((tok,), -9, dtype=torch.int32, device="cuda")
        self.top_p = torch.full((tok,), 0.9, device="cuda")
        qkv = self.qkv
        self.rope = rope_args(kind, qkv[:, :heads], self.q.view(tok, heads, dim), qkv[:, heads:heads + kv],
                              qkv[:, heads + kv:], self.kc, self.vc, self.pos, self.freq, dim, 0, 1.0, self.slot)
        self.tree = tree_args(kind, self.q, self.kc, self.vc, self.n_past, self.parent, self.att, dim ** -0.5)
        p = torch.Tensor.data_ptr
        self.pick = capi.SampleArgs(type=0, n_row=tok, n_vocab=vocab, row_stride=vocab, logits=p(self.logits),
                                    u=p(self.u), id=p(self.ids), top_p=p(self.top_p))

    def run(self):
        lib, st = capi.lib(), torch.cuda.current_stream().cuda_stream
        call(lib.sdy_rope_dev, self.rope, st)
        call(lib.sdy_tree_attention_dev, self.tree, st)
        torch.matmul(self.att.view(len(self.ids), -1).float(), self.w, out=self.logits)
        call(lib.sdy_sample_dev, self.pick, st)

    def check(self):
        heads, kv, dim = self.heads, self.kv, self.dim
        freq, pos = self.freq.cpu().numpy(), self.pos.cpu().numpy()
        close_rope(self.q.view(-1, heads, dim), self.qkv[:, :heads], self.pos, self.freq, 0, 1.0, self.kind)
        want_k, _ = ref.rope(f64(self.qkv[:, heads:heads + kv]), pos, freq, 0, 1.0)
        for s, past in enumerate(self.past):
            rows = slice(past, past + self.nodes)
            tok = slice(s * self.nodes, (s + 1) * self.nodes)
            np.testing.assert_allclose(f64(self.kc[s, :, rows]).transpose(1, 0, 2), want_k[tok], atol=0.04)
            assert torch.equal(self.vc[s, :, rows].transpose(0, 1), self.qkv[tok, heads + kv:])
            assert torch.equal(self.kc[s, :, :past], self.k0[s, :, :past])
            assert torch.equal(self.vc[s, :, past + self.nodes:], self.v0[s, :, past + self.nodes:])
        check_tree(self.kind, self.q, (f64(self.kc), f64(self.vc)), self.n_past, self.par, dim ** -0.5, self.att)
        x, u = f64(self.logits), f64(self.u)
        for r in range(len(x)):
            assert int(self.ids[r]) == ref.sample(x[r], u[r], top_p=float(np.float32(0.9)))[0]


@pytest.mark.parametrize("kind", KINDS)
def test_step_together(kind):
    step = Step(kind)
    step.run()
    torch.cuda.synchronize()
    step.check()


def test_step_on_another_stream_and_in_a_graph():
    """The step on a side stream, captured, and replayed on new inputs; a second step's graph replayed
    between, each with its own workspace."""
    steps = [Step("bf16", seed=1), Step("bf16", seed=2, past=(11, 300), nodes=7)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graphs = []
    with torch.cuda.stream(side):
        for step in steps:
            step.run()
        side.synchronize()
        for step in steps:
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side):
                step.run()
            graphs.append(graph)
    g = gen(99)
    for round_ in range(3):
        for step in steps:
            step.qkv.copy_(randn(g, *step.qkv.shape, kind="bf16"))
            step.u.copy_(torch.rand(len(step.u), generator=g, device="cuda"))
            step.att.fill_(float("nan"))
        torch.cuda.synchronize()
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for step in steps:
            step.check()


def test_step_lengths_change_between_replays():
    """The lengths are read on the device: a captured call serves a growing cache."""
    q, k, v, n_past, parent, par, clean = tree_case("bf16", 2, 6, 8, 2, 128, [900, 900], parents=True, poison=False)
    out = torch.empty_like(q)
    a = tree_args("bf16", q, k, v, n_past, parent, out, 0.1)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        call(capi.lib().sdy_tree_attention_dev, a, side.cuda_stream)
        side.synchronize()
        with torch.cuda.graph(graph, stream=side):
            call(capi.lib().sdy_tree_attention_dev, a, side.cuda_stream)
    for lengths in ([900, 0], [1, 65], [64, 899], [511, 640]):
        n_past.copy_(torch.tensor(lengths, dtype=torch.int32))
        out.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        check_tree("bf16", q, clean, n_past, par, 0.1, out)


def test_host_memory_is_refused():
    """Pageable host memory is refused before a launch; pinned memory works."""
    lib = capi.lib()
    x = torch.randn(2, 100)
    u = torch.rand(2, device="cuda")
    ids = torch.empty(2, dtype=torch.int32, device="cuda")
    p = torch.Tensor.data_ptr
    before = lib.sdy_kernel_launches()
    a = capi.SampleArgs(type=0, n_row=2, n_vocab=100, row_stride=100, logits=p(x), u=p(u), id=p(ids))
    assert lib.sdy_sample_dev(ctypes.byref(a), None) == -1 and "logits is not memory" in capi.last_error()
    lib.sdy_clear_error()
    q = torch.zeros(1, 1, 64)
    assert lib.sdy_rope_dev(ctypes.byref(rope_args("f32", q, q, None, None, None, None, u, u.double(), 64, 0)), None) == -1
    assert "is not memory" in capi.last_error() and lib.sdy_kernel_launches() == before
    lib.sdy_clear_error()
    pinned = x.pin_memory()
    got = torch.empty(2, dtype=torch.int32).pin_memory()
    a = capi.SampleArgs(type=0, n_row=2, n_vocab=100, row_stride=100, logits=p(pinned), u=p(u), id=p(got))
    call(lib.sdy_sample_dev, a)
    torch.cuda.synchronize()
    for r in range(2):
        assert int(got[r]) == ref.sample(f64(x[r]), float(u[r]))[0]


# ------------------------------------------------------------------------------------- the engine's sampled step

class Engine:
    """A context of a small random model through the library's own binding."""

    def __init__(self, path, max_seq=64):
        self.lib = capi.lib()
        err = ctypes.create_string_buffer(512)
        self.model = self.lib.engine_model_load(str(path).encode(), err, 512)
        assert self.model, err.value
        self.ctx = self.lib.engine_ctx_new(self.model, max_seq, 16, 0, 1, err, 512)
        assert self.ctx, err.value
        info = capi.EngineModelInfo()
        self.lib.engine_model_get_info(self.model, ctypes.byref(info))
        self.vocab = info.n_vocab

    def eval(self, tokens):
        assert self.lib.engine_eval(self.ctx, (ctypes.c_int32 * len(tokens))(*tokens), len(tokens)) == 0
        return np.ctypeslib.as_array(self.lib.engine_logits(self.ctx), (self.vocab,)).copy()

    def sample(self, tokens, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
        out = ctypes.c_int32(-5)
        rc = self.lib.sdy_engine_eval_sample(self.ctx, (ctypes.c_int32 * len(tokens))(*tokens), len(tokens), temperature,
                                             top_k, top_p, min_p, u, ctypes.byref(out))
        return rc, out.value

    def close(self):
        self.lib.engine_ctx_free(self.ctx)
        self.lib.engine_model_free(self.model)


@pytest.fixture(scope="module")
def model_path(tmp_path_factory):
    from sardyne_b200 import synth
    return synth.write_model(tmp_path_factory.mktemp("model") / "m.gguf",
                             synth.Spec(dim=256, head_dim=64, ffn=512, vocab=1500, context=64, kinds="Q8_0", seed=4))


def test_engine_eval_sample(model_path):
    """Tokens sampled on the device are those sampled from the logits that a second context returns
    for the same tokens, prompts in one and several chunks, then step by step."""
    a, b = Engine(model_path), Engine(model_path)
    rng = np.random.default_rng(5)
    tokens = [int(t) for t in rng.integers(0, a.vocab, 37)]
    settings = [dict(), dict(temperature=0.7, top_k=40, top_p=0.95), dict(temperature=0.0), dict(min_p=0.1),
                dict(temperature=1.3, top_p=0.6), dict(temperature=2.0, top_k=3)]
    for step in range(12):
        how, u = settings[step % len(settings)], float(np.float32(rng.random()))
        logits = a.eval(tokens)
        rc, got = b.sample(tokens, u, **how)
        assert rc == 0 and not b.lib.engine_logits(b.ctx) and b.lib.engine_n_past(b.ctx) == a.lib.engine_n_past(a.ctx)
        f32 = {k: float(np.float32(v)) if isinstance(v, float) else v for k, v in how.items()}
        assert got == ref.sample(logits.astype(np.float64), u, **f32)[0], how
        tokens = [got]
    assert b.sample([a.vocab], 0.5)[0] == -1 and b.lib.engine_n_past(b.ctx) == a.lib.engine_n_past(a.ctx)
    assert b.lib.sdy_engine_eval_sample(b.ctx, (ctypes.c_int32 * 1)(1), 1, 1.0, 0, 1.0, 0.0, 0.5, None) == -1
    assert np.array_equal(a.eval([3]), b.eval([3]))
    a.close()
    b.close()


def test_engine_eval_sample_without_valid_logits(tmp_path):
    from sardyne_b200 import synth
    path = synth.write_model(tmp_path / "nan.gguf", synth.Spec(norm_noise=float("nan")))
    e = Engine(path, 16)
    rc, _ = e.sample([1, 2], 0.5)
    assert rc == -1 and e.lib.engine_n_past(e.ctx) == 0 and e.lib.engine_last_error(e.ctx)
    e.close()
