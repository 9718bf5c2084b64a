"""Refusals of the shared-prefix calls that need no GPU."""
import ctypes as C

import numpy as np
import pytest

from embedcuda import _lib, model


def test_needs_init():
    L = _lib.lib()
    ids = np.array([1, 2], np.int32)
    offs = np.array([0, 2], np.int64)
    out = np.empty((1, 8), np.float32)
    p = C.c_int(0)
    if L.ec_device_count() == 0:
        assert L.ec_prefix_open(_lib.ptr(ids, C.c_int32), 2, C.byref(p)) == _lib.EC_ESTATE
        assert L.ec_prefix_close(1) == _lib.EC_ESTATE
        assert L.ec_embed_batch_prefix(1, _lib.ptr(ids, C.c_int32), _lib.ptr(offs, C.c_int64), 1,
                                       _lib.ptr(out, C.c_float), 8) == _lib.EC_ESTATE
    else:
        assert L.ec_prefix_open(None, 2, C.byref(p)) == _lib.EC_EINVAL
        assert L.ec_prefix_close(1 << 30) == _lib.EC_EINVAL


def test_prefix_is_a_vector():
    with pytest.raises(ValueError):
        model.Prefix(np.zeros((2, 2), np.int32))
