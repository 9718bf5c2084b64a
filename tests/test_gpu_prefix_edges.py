"""Shared prefixes and Llama models at the edges: waits that gave up, what
config.json and earlier uploads say.  Models, helpers and tolerances are those
of test_gpu_prefix.py."""
import ctypes as C
import dataclasses
import json
import os

import numpy as np
import pytest

from embedcuda import _lib, model, synth
from test_gpu_prefix import COS, LLAMA64, QWEN, _batch, _cos, _ids, _load

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("shape", [QWEN, LLAMA64], ids=lambda s: s.name)
def test_a_callers_time_out_is_not_the_librarys(synth_root, ec, shape):
    """The mark of a caller's own operator neither fails an embedding nor is
    cleared by one."""
    _load(synth_root, shape)
    rng = np.random.default_rng(3)
    ids, offs = _batch(rng, shape, [3, 17, 130])
    L = ec.lib()
    assert L.ec_op_status() == 0
    with model.Prefix(_ids(rng, shape, 40)) as p:
        want, plain = p.embed_batch(ids, offs), model.embed_batch(ids, offs)
        assert L.ecdbg_op_timeout() == 0
        assert np.array_equal(p.embed_batch(ids, offs), want)
        assert np.array_equal(model.embed_batch(ids, offs), plain)
        with model.Prefix(_ids(rng, shape, 3)) as other:
            other.embed_batch(ids, offs)
        assert L.ec_op_status() == _lib.EC_ETIMEOUT
        assert L.ec_op_status() == 0
        assert np.array_equal(p.embed_batch(ids, offs), want)


def test_a_forward_that_timed_out_leaves_the_next_ones_right(synth_root, ec):
    """Texts of few tokens behind a long prefix: more tiles than SMs, so some
    are cut and joined by the workspace's counts."""
    _load(synth_root, QWEN)
    rng = np.random.default_rng(8)
    batches = [_batch(rng, QWEN, rng.integers(1, 9, 120)) for _ in range(2)]
    with model.Prefix(_ids(rng, QWEN, 1000)) as p, model.Prefix(_ids(rng, QWEN, 900)) as other:
        want = [x.embed_batch(*b) for x in (p, other) for b in batches]
        for _ in range(2):
            assert ec.lib().ecdbg_prefix_timeout() == 0
            with pytest.raises(_lib.EcError) as e:
                p.embed_batch(*batches[1])
            assert e.value.code == _lib.EC_ETIMEOUT
            for _ in range(2):
                got = [x.embed_batch(*b) for x in (p, other) for b in batches]
                for g, w in zip(got, want):
                    assert np.array_equal(g, w)


def _upload(name, dims, raw):
    dims, raw = np.array(dims, np.int64), np.ascontiguousarray(raw)
    _lib.check(_lib.lib().ec_upload_tensor(name.encode(), _lib.EC_BF16, dims.ctypes.data_as(C.POINTER(C.c_int64)),
                                           len(dims), raw.ctypes.data, raw.nbytes))


def _assemble(d, **changes):
    """ec_load_model of what is uploaded, config.json changed."""
    with open(os.path.join(d, "config.json")) as f:
        cfg = {**json.load(f), **changes}
    fam, dim = C.c_int(0), C.c_int(0)
    _lib.check(_lib.lib().ec_load_model(json.dumps(cfg).encode(), None, C.byref(fam), C.byref(dim)))


def test_a_qwen3_models_norms_stay(synth_root, ec):
    """All weights but the q/k norms uploaded again: a Qwen3 model keeps them."""
    qwen = synth.with_layers(dataclasses.replace(synth.QWEN3_06B, name="qwen-norms"), 1, vocab=2048)
    d = _load(synth_root, qwen)
    ids, offs = _batch(np.random.default_rng(4), qwen, [5, 70])
    want = model.embed_batch(ids, offs)
    for name, (dtype, dims, raw) in synth.make_weights(qwen, 3).items():
        if not name.endswith(("q_norm.weight", "k_norm.weight")):
            _upload(name, dims, raw)
    _assemble(d)
    assert np.array_equal(model.embed_batch(ids, offs), want)


# ------------------------------------------------------- scaled frequencies --
def _frequencies(hd, theta, s):
    """Turns per position of a head's pairs, and the tables' amplitude."""
    i = np.arange(hd // 2)
    f, amp, kind = theta ** (-2.0 * i / hd), 1.0, (s or {}).get("rope_type", (s or {}).get("type"))
    if kind == "linear":
        f = f / s["factor"]
    if kind == "llama3":
        turns = s["original_max_position_embeddings"] * f / (2 * np.pi)
        low, high = s["low_freq_factor"], s["high_freq_factor"]
        keep = np.clip((turns - low) / (high - low), 0, 1)
        f = (1 - keep) * f / s["factor"] + keep * f
    if kind == "yarn":
        n = s["original_max_position_embeddings"]
        at = lambda b: hd * np.log(n / (b * 2 * np.pi)) / (2 * np.log(theta))  # noqa: E731
        lo, hi = max(np.floor(at(s.get("beta_fast", 32))), 0), min(np.ceil(at(s.get("beta_slow", 1))), hd - 1)
        r = np.clip((i - lo) / max(hi - lo, 1e-3), 0, 1)
        f = f / s["factor"] * r + f * (1 - r)
        amp = s.get("attention_factor") or 0.1 * np.log(s["factor"]) + 1
    return f, amp


def _weights(shape, seed):
    """The synthetic weights, queries eight times as large: with scores that far
    apart the angles count."""
    w = synth.make_weights(shape, seed)
    for name, (dtype, dims, raw) in w.items():
        if name.endswith("q_proj.weight"):
            w[name] = dtype, dims, synth.f32_to_bf16_bits((raw.astype(np.uint32) << 16).view(np.float32) * 8)
    return w


def _llama(shape, seed, ids, scaling):
    """Last token's unit vector of a Llama model, in 64 bits."""
    w = {name: (raw.astype(np.uint32) << 16).view(np.float32).reshape(dims).astype(np.float64)
         for name, (_, dims, raw) in _weights(shape, seed).items()}
    hd, hq, hk, n = shape.head_dim, shape.heads, shape.kv_heads, len(ids)
    f, amp = _frequencies(hd, shape.rope_theta, scaling)
    a = np.outer(np.arange(n), f)[:, None]
    c, s = amp * np.cos(a), amp * np.sin(a)
    norm = lambda x, g: x / np.sqrt((x * x).mean(-1, keepdims=True) + shape.rms_eps) * g  # noqa: E731

    def turn(x):
        lo, hi = x[..., :hd // 2], x[..., hd // 2:]
        return np.concatenate([lo * c - hi * s, hi * c + lo * s], -1)
    h = w["embed_tokens.weight"][ids]
    for li in range(shape.layers):
        p = lambda x: w[f"layers.{li}.{x}.weight"]  # noqa: E731,B023
        x = norm(h, p("input_layernorm"))
        q, k, v = ((x @ p(f"self_attn.{y}_proj").T).reshape(n, -1, hd) for y in "qkv")
        q, k, v = turn(q), turn(k).repeat(hq // hk, 1), v.repeat(hq // hk, 1)
        z = np.where(np.tril(np.ones((n, n), bool)), np.einsum("mhd,nhd->hmn", q, k) / np.sqrt(hd), -np.inf)
        z = np.exp(z - z.max(-1, keepdims=True))
        o = np.einsum("hmn,nhd->mhd", z / z.sum(-1, keepdims=True), v).reshape(n, -1)
        h = h + o @ p("self_attn.o_proj").T
        x = norm(h, p("post_attention_layernorm"))
        g = x @ p("mlp.gate_proj").T
        h = h + (g / (1 + np.exp(-g)) * (x @ p("mlp.up_proj").T)) @ p("mlp.down_proj").T
    y = norm(h, w["norm.weight"])[-1]
    return y / np.linalg.norm(y)


SCALINGS = [None, {"rope_type": "default"}, {"type": "linear", "factor": 16.0},
            {"rope_type": "llama3", "factor": 32.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0,
             "original_max_position_embeddings": 64},
            {"rope_type": "yarn", "factor": 16.0, "original_max_position_embeddings": 64, "attention_factor": 1.5},
            {"type": "yarn", "factor": 8.0, "beta_fast": 4.0, "beta_slow": 2.0, "original_max_position_embeddings": 128}]


@pytest.mark.parametrize("scaling", SCALINGS, ids=lambda s: str((s or {}).get("rope_type", (s or {}).get("type"))))
def test_scaled_frequencies(synth_root, ec, scaling):
    """Another head dim than 128: the frequencies are config.json's."""
    shape = dataclasses.replace(LLAMA64, name="llama-scaled", vocab=512)
    d = _load(synth_root, shape)
    ids, offs = _batch(np.random.default_rng(9), shape, [7, 40, 300])
    for name, (_, dims, raw) in _weights(shape, 3).items():
        if name.endswith("q_proj.weight"):
            _upload(name, dims, raw)
    _assemble(d, rope_scaling=scaling)
    got = model.embed_batch(ids, offs)
    want, plain = (np.stack([_llama(shape, 3, ids[a:b], s) for a, b in zip(offs, offs[1:])]) for s in (scaling, None))
    assert _cos(got, want).min() >= COS, _cos(got, want)
    if scaling and "factor" in scaling:  # the plain frequencies' are further away
        assert _cos(want, plain).max() < 1 - 4 * (1 - COS)


def test_scaled_frequencies_refusals(synth_root, ec):
    d = _load(synth_root, dataclasses.replace(LLAMA64, name="llama-scaled", vocab=512))
    for bad, code in (({"rope_type": "longrope"}, _lib.EC_EUNSUPPORTED), ({"factor": 2.0}, _lib.EC_EINVAL),
                      ({"rope_type": "linear"}, _lib.EC_EINVAL), ({"rope_type": "llama3", "factor": 8.0}, _lib.EC_EINVAL),
                      ({"rope_type": "yarn", "factor": 8.0, "truncate": False}, _lib.EC_EUNSUPPORTED),
                      ({"rope_type": "yarn", "factor": 8.0, "mscale": 0.7}, _lib.EC_EUNSUPPORTED)):
        with pytest.raises(_lib.EcError) as e:
            _assemble(d, rope_scaling=bad)
        assert e.value.code == code, bad
    _assemble(d, rope_scaling={"rope_type": "dynamic", "factor": 4.0})
    _assemble(d, rope_scaling={"rope_type": "yarn", "factor": 8.0})  # from max_position_embeddings


def test_head_dim_128_keeps_its_table(synth_root, ec):
    d = _load(synth_root, QWEN)
    ids, offs = _batch(np.random.default_rng(2), QWEN, [3, 100])
    want = model.embed_batch(ids, offs)
    _assemble(d, rope_scaling={"rope_type": "yarn", "factor": 4.0, "original_max_position_embeddings": 64})
    assert np.array_equal(model.embed_batch(ids, offs), want)
