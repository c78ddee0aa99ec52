"""The drafted-token operators' host side, without a GPU: the frequencies of the scaled rotary
positions, and the refusal of arguments that the kernels do not take (before any CUDA call)."""
import ctypes

import numpy as np
import pytest

import drafted_ref as ref
from sardyne_b200 import capi

SPECS = [dict(n_rot=128, theta=1e6), dict(n_rot=2, theta=1e4), dict(n_rot=64, theta=5e5, scaling=1, factor=4.0),
         dict(n_rot=128, theta=5e5, scaling=2, factor=8.0, low=1.0, high=4.0, orig_ctx=8192),
         dict(n_rot=128, theta=1e6, scaling=3, factor=4.0, low=1.0, high=32.0, orig_ctx=32768),
         dict(n_rot=96, theta=1e4, scaling=3, factor=16.0, low=1.0, high=32.0, orig_ctx=4096),
         dict(n_rot=10, theta=1.5, scaling=3, factor=2.0, low=1.0, high=2.0, orig_ctx=1)]


def freqs(factors=None, **kw):
    spec = capi.RopeSpec(**kw)
    if factors is not None:
        factors = np.ascontiguousarray(factors, np.float32)
        spec.factors = factors.ctypes.data
    out = np.full(max(kw["n_rot"], 2) // 2, np.nan)
    rc = capi.lib().sdy_rope_freqs(ctypes.byref(spec), out.ctypes.data_as(ctypes.POINTER(ctypes.c_double)))
    return rc, out


@pytest.mark.parametrize("spec", SPECS)
def test_rope_freqs(spec):
    rc, got = freqs(**spec)
    assert rc == 0
    # pow, log and a handful of roundings; the ramps of scaling 2 and 3 multiply them by at most
    # 1/(high - low) and the number of turns
    np.testing.assert_allclose(got, ref.rope_freqs(**spec), rtol=1e-12)
    factors = np.linspace(1, 7, spec["n_rot"] // 2, dtype=np.float32)
    rc, got = freqs(factors=factors, **spec)
    assert rc == 0
    np.testing.assert_allclose(got, ref.rope_freqs(factors=factors, **spec), rtol=1e-12)


def test_rope_freqs_keeps_and_stretches_the_ends():
    """By wavelength: fast pairs are untouched, slow ones divided by the factor, exactly."""
    _, plain = freqs(n_rot=128, theta=5e5)
    _, got = freqs(n_rot=128, theta=5e5, scaling=2, factor=8.0, low=1.0, high=4.0, orig_ctx=8192)
    turns = 8192 * plain / (2 * np.pi)
    assert np.array_equal(got[turns > 4], plain[turns > 4]) and np.array_equal(got[turns < 1], plain[turns < 1] / 8)
    assert (np.diff(got) < 0).all()


@pytest.mark.parametrize("change,word", [
    (dict(n_rot=3), "n_rot"), (dict(n_rot=0), "n_rot"), (dict(n_rot=2048), "n_rot"), (dict(scaling=4), "scaling"),
    (dict(scaling=-1), "scaling"), (dict(theta=0.0), "theta"), (dict(theta=float("nan")), "theta"),
    (dict(factor=0.0), "factor"), (dict(factor=float("inf")), "factor"), (dict(orig_ctx=0), "orig_ctx"),
    (dict(low=0.0), "low"), (dict(high=1.0), "low"), (dict(scaling=3, theta=1.0), "theta > 1"),
    (dict(factors=np.zeros(64)), "factors")])
def test_rope_freqs_refusals(change, word):
    rc, out = freqs(**{**dict(n_rot=128, theta=1e4, scaling=2, factor=2.0, low=1.0, high=4.0, orig_ctx=64), **change})
    assert rc == -1 and word in capi.last_error() and np.isnan(out).all()
    capi.lib().sdy_clear_error()
    assert capi.lib().sdy_rope_freqs(None, None) == -1
    capi.lib().sdy_clear_error()


P = 4096  # stands for a device pointer: these calls end before any is looked at


def rope_args(**kw):
    base = dict(type=0, n_tok=2, n_head=4, n_kv_head=2, head_dim=64, n_rot=64, mscale=1.0, freq=P, pos=P, q=P,
                q_tok=256, q_head=64, q_out=2 * P, q_out_tok=256, q_out_head=64, k=P, k_tok=128, k_head=64, v=P,
                v_tok=128, v_head=64, k_cache=3 * P, v_cache=4 * P, n_seq=1, max_seq=16, cache_seq=2048,
                cache_head=1024, cache_row=64)
    return capi.RopeArgs(**{**base, **kw})


def refused(fn, args, word):
    lib = capi.lib()
    lib.sdy_clear_error()
    before = lib.sdy_kernel_launches()
    assert fn(None if args is None else ctypes.byref(args), None) == -1
    assert word in capi.last_error(), capi.last_error()
    assert lib.sdy_kernel_launches() == before
    lib.sdy_clear_error()


@pytest.mark.parametrize("change,word", [
    (dict(type=8), "type"), (dict(n_tok=-1), "counts"), (dict(n_head=-1), "counts"), (dict(head_dim=0), "head_dim"),
    (dict(head_dim=1025), "head_dim"), (dict(n_rot=63), "n_rot"), (dict(n_rot=66), "n_rot"), (dict(n_rot=-2), "n_rot"),
    (dict(mscale=float("nan")), "mscale"), (dict(freq=0), "freq"), (dict(pos=0), "pos"), (dict(q=0), "q"),
    (dict(q_out=0), "q_out"), (dict(k=0), "k or"), (dict(k_cache=0), "k or"), (dict(v_cache=0), "k or"),
    (dict(n_seq=0), "no rows"), (dict(max_seq=0), "no rows"), (dict(q_tok=-256), "negative"),
    (dict(q_out_tok=64), "q_out overlap"), (dict(q_out_head=32), "q_out overlap"), (dict(cache_row=32), "cache overlap"),
    (dict(cache_head=64), "cache overlap"), (dict(n_seq=2, cache_seq=0), "cache overlap"),
    (dict(q_out=P, q_out_tok=512), "in place"), (dict(q=P + 2), "aligned"), (dict(freq=P + 4), "aligned"),
    (dict(slot=P + 4), "aligned")])
def test_rope_refusals(change, word):
    refused(capi.lib().sdy_rope_dev, rope_args(**change), word)


def tree_args(**kw):
    base = dict(type=30, n_seq=2, n_node=8, n_head=4, n_kv_head=2, head_dim=64, max_seq=100, scale=0.125, q=P,
                q_seq=2048, q_node=256, q_head=64, k_cache=2 * P, v_cache=3 * P, cache_seq=12800, cache_head=6400,
                cache_row=64, n_past=P, parent=P, out=4 * P, out_seq=2048, out_node=256, out_head=64, ws=5 * P,
                ws_bytes=1 << 30)
    return capi.TreeAttentionArgs(**{**base, **kw})


@pytest.mark.parametrize("change,word", [
    (dict(type=12), "type"), (dict(n_seq=-1), "n_seq"), (dict(n_seq=65536), "n_seq"), (dict(n_node=0), "n_node"),
    (dict(n_node=257), "n_node"), (dict(n_head=3), "multiple"), (dict(n_kv_head=0), "multiple"),
    (dict(n_head=0), "multiple"), (dict(head_dim=60), "head_dim"), (dict(head_dim=264), "head_dim"),
    (dict(head_dim=0), "head_dim"), (dict(max_seq=0), "no rows"), (dict(scale=float("inf")), "scale"),
    (dict(q=0), "missing"), (dict(k_cache=0), "missing"), (dict(n_past=0), "missing"), (dict(out=0), "missing"),
    (dict(q=P + 8), "aligned"), (dict(out=4 * P + 2), "aligned"), (dict(n_past=P + 2), "aligned"),
    (dict(q_node=-256), "negative"), (dict(cache_row=68), "16 bytes"), (dict(out_head=68), "16 bytes"),
    (dict(out_node=64), "overlap"), (dict(out_head=56), "overlap"), (dict(out=P), "out is q"),
    (dict(ws=0), "ws missing"), (dict(ws_bytes=0), "ws missing")])
def test_tree_attention_refusals(change, word):
    if "ws" in change or "ws_bytes" in change:  # a shape that is split over the keys and needs a workspace
        change = dict(change, max_seq=1 << 20, cache_head=1 << 26, cache_seq=1 << 27)
    refused(capi.lib().sdy_tree_attention_dev, tree_args(**change), word)


def test_tree_attention_bytes():
    lib = capi.lib()
    for shape in (dict(), dict(head_dim=256, q_head=256, out_head=256), dict(type=0), dict(n_head=40, n_node=200)):
        need = lib.sdy_tree_attention_bytes(ctypes.byref(tree_args(**shape)))
        assert need == lib.sdy_tree_attention_bytes(ctypes.byref(tree_args(**{**shape, "cache_seq": 0, "q": 0, "ws": 0, "max_seq": 7})))
    assert lib.sdy_tree_attention_bytes(ctypes.byref(tree_args(max_seq=1 << 20))) > 0
    assert lib.sdy_tree_attention_bytes(ctypes.byref(tree_args(n_node=300))) == 0 and "n_node" in capi.last_error()
    lib.sdy_clear_error()


def sample_args(**kw):
    base = dict(type=0, n_row=2, n_vocab=1000, row_stride=1000, logits=P, u=P, id=P, prob=P)
    return capi.SampleArgs(**{**base, **kw})


@pytest.mark.parametrize("change,word", [
    (dict(type=2), "type"), (dict(n_row=-1), "counts"), (dict(n_vocab=0), "n_vocab"), (dict(n_vocab=400001), "n_vocab"),
    (dict(row_stride=-1), "negative"), (dict(logits=0), "missing"), (dict(u=0), "missing"), (dict(id=0), "missing"),
    (dict(logits=P + 2), "aligned"), (dict(top_k=P + 1), "aligned")])
def test_sample_refusals(change, word):
    refused(capi.lib().sdy_sample_dev, sample_args(**change), word)


def test_no_argument_block_and_counts_of_zero():
    lib = capi.lib()
    for fn, args, zero in ((lib.sdy_rope_dev, rope_args, "n_tok"), (lib.sdy_tree_attention_dev, tree_args, "n_seq"),
                           (lib.sdy_sample_dev, sample_args, "n_row")):
        refused(fn, None, "no argument block")
        before = lib.sdy_kernel_launches()
        assert fn(ctypes.byref(args(**{zero: 0})), None) == 0 and lib.sdy_kernel_launches() == before
    assert lib.sdy_engine_eval_sample(None, None, 0, 1.0, 0, 1.0, 0.0, 0.5, None) == -1
