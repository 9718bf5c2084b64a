"""Texts behind a shared prefix, and Llama head dims other than 128: against
the CPU oracle on prefix + text, and against embed_batch of prefix + text.

Tolerance: the cosine bound of the BF16 models against the oracle, 0.999 (an
angle a with 1 - cos a = 0.001); two results within that angle of the oracle
are within 2a of each other, and 1 - cos 2a <= 4 (1 - cos a) = 0.004.
"""
import os

import numpy as np
import pytest

from embedcuda import _lib, model, synth
from oracle import oracle

pytestmark = pytest.mark.gpu

COS = 0.999
COS_PAIR = 0.996

QWEN = synth.with_layers(synth.QWEN3_06B, 2, vocab=4096)
LLAMA64 = synth.ModelShape("llama-hd64", "llama", 512, 2, 8, 1024, 2048, 1024, "BF16", "last",
                           kv_heads=2, head_dim=64, rope_theta=10000.0, rms_eps=1e-5)
LLAMA96 = synth.ModelShape("llama-hd96", "llama", 512, 2, 4, 1024, 2048, 1024, "BF16", "last",
                           kv_heads=2, head_dim=96, rope_theta=500000.0, rms_eps=1e-5)
LLAMA16 = synth.ModelShape("llama-hd16", "llama", 256, 2, 8, 512, 2048, 1024, "F32", "last",
                           kv_heads=8, head_dim=16, rope_theta=10000.0, rms_eps=1e-5)
SHAPES = {s.name: s for s in (QWEN, LLAMA64, LLAMA96, LLAMA16)}


def _cos(a, b):
    return np.sum(a * b, axis=1) / (np.linalg.norm(a, axis=1) * np.linalg.norm(b, axis=1))


def _load(synth_root, shape):
    d = synth.build_model_dir(shape, 3, synth_root)
    assert model.load_model(d) == "llama"
    return d


def _ids(rng, shape, n):
    return rng.integers(0, shape.vocab, n).astype(np.int32)


def _batch(rng, shape, lengths):
    offs = np.zeros(len(lengths) + 1, np.int64)
    offs[1:] = np.cumsum(lengths)
    return _ids(rng, shape, int(offs[-1])), offs


def _joined(prefix, ids, offs):
    parts = [np.concatenate([prefix, ids[offs[s]:offs[s + 1]]]) for s in range(len(offs) - 1)]
    o = np.zeros(len(offs), np.int64)
    o[1:] = np.cumsum([p.size for p in parts])
    return np.concatenate(parts).astype(np.int32), o


def _oracle(d, ids, offs):
    n = len(offs) - 1
    return oracle.OracleModel(d).embed_batch(ids, offs, threads=n,
                                             seq_threads=max(1, (os.cpu_count() or 1) // n))


@pytest.mark.parametrize("name", ["llama-hd64", "llama-hd96", "llama-hd16"])
def test_other_head_dims(synth_root, ec, name):
    shape = SHAPES[name]
    d = _load(synth_root, shape)
    ids, offs = _batch(np.random.default_rng(1), shape, [1, 2, 40, 129, 300])
    got = model.embed_batch(ids, offs)
    cos = _cos(got, _oracle(d, ids, offs))
    assert cos.min() >= COS, cos


@pytest.mark.parametrize("name", sorted(SHAPES))
@pytest.mark.parametrize("n", [1, 31, 32, 33, 100])
def test_prefix_against_oracle(synth_root, ec, name, n):
    shape = SHAPES[name]
    d = _load(synth_root, shape)
    rng = np.random.default_rng(n)
    prefix = _ids(rng, shape, n)
    ids, offs = _batch(rng, shape, [1, 2, 31, 65, 150])
    whole = _joined(prefix, ids, offs)
    with model.Prefix(prefix) as p:
        got = p.embed_batch(ids, offs)
        assert np.array_equal(got, p.embed_batch(ids, offs))  # replayed
        one = np.stack([p.embed(ids[offs[s]:offs[s + 1]]) for s in range(2)])
    cos = _cos(got, _oracle(d, *whole))
    assert cos.min() >= COS, cos
    assert _cos(one, got[:2]).min() >= COS_PAIR
    assert _cos(got, model.embed_batch(*whole)).min() >= COS_PAIR


@pytest.mark.parametrize("count,longest,n", [(1300, 20, 7), (700, 200, 64), (90, 900, 120)])
def test_many_texts(synth_root, ec, count, longest, n):
    """More texts and tokens than one forward takes."""
    _load(synth_root, QWEN)
    rng = np.random.default_rng(count)
    prefix = _ids(rng, QWEN, n)
    ids, offs = _batch(rng, QWEN, rng.integers(1, longest + 1, count))
    with model.Prefix(prefix) as p:
        got = p.embed_batch(ids, offs)
    assert np.isfinite(got).all()
    assert _cos(got, model.embed_batch(*_joined(prefix, ids, offs))).min() >= COS_PAIR


def test_several_prefixes(synth_root, ec):
    """Prefixes side by side, closed and opened again, the same lengths behind
    each (captured forwards must not be mixed up)."""
    _load(synth_root, QWEN)
    rng = np.random.default_rng(5)
    ids, offs = _batch(rng, QWEN, [3, 17, 30])
    prefixes = [_ids(rng, QWEN, n) for n in (5, 40, 64, 5, 5, 96, 2, 9, 11)]
    want = [model.embed_batch(*_joined(p, ids, offs)) for p in prefixes]
    opened = [model.Prefix(p) for p in prefixes[:8]]
    first = [p.embed_batch(ids, offs) for p in opened]
    for f, w in zip(first, want):
        assert _cos(f, w).min() >= COS_PAIR
    with pytest.raises(RuntimeError):
        model.Prefix(prefixes[8])
    stale = opened[3]._id
    opened[3].close()
    with model.Prefix(prefixes[8]) as again:  # in the closed one's place
        assert _cos(again.embed_batch(ids, offs), want[8]).min() >= COS_PAIR
        for k in (0, 1, 2, 4, 7):
            assert np.array_equal(opened[k].embed_batch(ids, offs), first[k])
        bad = model.Prefix.__new__(model.Prefix)
        bad._id = stale
        with pytest.raises(RuntimeError):
            bad.embed_batch(ids, offs)
    for k in (0, 1, 2, 4, 5, 6, 7):
        opened[k].close()
    plain = model.embed_batch(ids, offs)  # without a prefix, as ever
    assert np.array_equal(plain, model.embed_batch(ids, offs))


def test_prefix_limits(synth_root, ec):
    _load(synth_root, QWEN)
    rng = np.random.default_rng(6)
    with pytest.raises(RuntimeError):
        model.Prefix(_ids(rng, QWEN, 0))
    with pytest.raises(RuntimeError):
        model.Prefix(_ids(rng, QWEN, 1024))
    with pytest.raises(RuntimeError):
        model.Prefix(np.array([QWEN.vocab], np.int32))
    prefix, text = _ids(rng, QWEN, 1023), _ids(rng, QWEN, 2)
    with model.Prefix(prefix) as p:
        got = p.embed(text[:1])
        with pytest.raises(RuntimeError):
            p.embed(text)
        with pytest.raises(RuntimeError):
            p.embed(text[:0])
        with pytest.raises(RuntimeError):
            p.embed(np.array([-1], np.int32))
        assert np.array_equal(got, p.embed(text[:1]))
    want = model.embed(np.concatenate([prefix, text[:1]]))
    assert _cos(got[None], want[None])[0] >= COS_PAIR
    p = model.Prefix(prefix)
    _load(synth_root, QWEN)  # ends the prefixes of the model before
    with pytest.raises(RuntimeError):
        p.embed(text[:1])
    with pytest.raises(RuntimeError):
        p.close()


def test_prefix_needs_causal(synth_root, ec):
    d = synth.build_model_dir(synth.with_layers(synth.MINILM, 2), 0, synth_root)
    model.load_model(d)
    with pytest.raises(RuntimeError):
        model.Prefix(np.array([101, 2000], np.int32))


def test_head_dim_refusals(synth_root, ec):
    import dataclasses
    for bad in (dict(name="llama-hd20", head_dim=20), dict(name="llama-hd136", head_dim=136),
                dict(name="qwen3-hd64", model_type="qwen3", head_dim=64)):
        d = synth.build_model_dir(dataclasses.replace(LLAMA64, **bad), 3, synth_root)
        with pytest.raises(RuntimeError) as e:
            model.load_model(d)
        assert "head_dim" in str(e.value)


def test_norms_of_an_earlier_model(synth_root, ec):
    """A Llama model without q/k norms after one with them does not take
    theirs; weights of a layer uploaded again keep the layer's norms."""
    import dataclasses
    qwen = synth.with_layers(dataclasses.replace(synth.QWEN3_06B, name="qwen-norms"), 1, vocab=2048)
    plain = dataclasses.replace(qwen, name="llama-no-norms", model_type="llama")
    ids, offs = _batch(np.random.default_rng(4), qwen, [5, 70])
    d = _load(synth_root, plain)
    first = model.embed_batch(ids, offs)
    assert _cos(first, _oracle(d, ids, offs)).min() >= COS
    dq = _load(synth_root, qwen)
    normed = model.embed_batch(ids, offs)
    assert _cos(normed, _oracle(dq, ids, offs)).min() >= COS
    # one weight again, and the model put together anew: the same model
    w = synth.make_weights(qwen, 3)["layers.0.self_attn.q_proj.weight"]
    dims = np.array(w[1], np.int64)
    import ctypes as C
    raw = np.ascontiguousarray(w[2])
    _lib.check(_lib.lib().ec_upload_tensor(b"layers.0.self_attn.q_proj.weight", _lib.EC_BF16,
                                           dims.ctypes.data_as(C.POINTER(C.c_int64)), 2, raw.ctypes.data, raw.nbytes))
    with open(os.path.join(dq, "config.json")) as f:
        cfg = f.read()
    fam, dim = C.c_int(0), C.c_int(0)
    _lib.check(_lib.lib().ec_load_model(cfg.encode(), None, C.byref(fam), C.byref(dim)))
    assert np.array_equal(model.embed_batch(ids, offs), normed)
    _load(synth_root, plain)
    assert np.array_equal(model.embed_batch(ids, offs), first)
