"""Shared prefixes and Llama models at the edges: waits that gave up, what
config.json and earlier uploads say.  Models, helpers and tolerances are those
of test_gpu_prefix.py."""
import numpy as np
import pytest

from embedcuda import _lib, model
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
