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
from test_gpu_prefix import LLAMA64, QWEN, _batch, _ids, _load

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
