"""Refusals of the operators on device buffers at the edges of their ranges;
none of these calls needs a GPU (pointers are never followed)."""
import os
import subprocess
import sys

import pytest
import torch

from conftest import REPO
from embedcuda import _lib, ops
from test_ops import L, open_, refused


def test_work_size_of_more_heads_than_a_tile_has_rows():
    """In a process of its own: a division by zero would end this one."""
    code = ("import sys, os, ctypes as C; sys.path[:0] = [%r, os.path.join(%r, 'lisp-embed_b200'), %r];"
            "from test_ops import L, open_; rc, h = open_(heads=1); assert rc == 0;"
            "print([L().ec_attn_cached_work_size(h, 4, q, 1, 4) for q in (129, 256, 1024, 2048, 1 << 30)])"
            ) % (REPO, REPO, os.path.join(REPO, "tests"))
    out = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert out.returncode == 0, (out.returncode, out.stderr)
    assert out.stdout.strip() == str([_lib.EC_EINVAL] * 5)


def test_work_size_takes_what_the_call_takes():
    for heads, most in ((1, 128), (4, 512), (16, 1024)):
        rc, h = open_(heads=heads)
        assert rc == 0
        assert L().ec_attn_cached_work_size(h, 4, most, 1, 4) > 0
        refused(L().ec_attn_cached_work_size(h, 4, most + heads, 1, 4), "query heads")
        refused(L().ec_attn_cached_work_size(h, 4, 0, 1, 4), "query heads")
        if heads > 1:
            refused(L().ec_attn_cached_work_size(h, 4, most - 1, 1, 4), "query heads")
        refused(L().ec_attn_cached_work_size(h, -1, most, 1, 4), "shape")
        assert L().ec_kv_close(h) == 0


@pytest.mark.parametrize("scaling,text", [
    ({"rope_type": "yarn", "factor": 4.0, "original_max_position_embeddings": 4096, "truncate": False}, "truncate"),
    ({"rope_type": "yarn", "factor": 4.0, "original_max_position_embeddings": 4096, "mscale": 0.707,
      "mscale_all_dim": 0.7}, "mscale, mscale_all_dim"),
    ({"rope_type": "llama3", "factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0,
      "original_max_position_embeddings": 8192, "short_factor": [1.0]}, "short_factor"),
    ({"rope_type": "linear", "factor": 4.0, "rope_theta": 1e6}, "rope_theta"),
])
def test_rope_scaling_that_would_be_dropped(scaling, text):
    cos = torch.zeros(16, 32)
    with pytest.raises(ValueError, match=text):
        ops.rope_table(cos, cos, 1e4, scaling, stream=0)


@pytest.mark.parametrize("scaling", [
    {"rope_type": "default", "rope_theta": 1e4, "factor": 4.0}, {"rope_type": "linear", "factor": 4.0, "beta_fast": 32},
    {"type": "yarn", "factor": 4.0, "original_max_position_embeddings": 4096, "finetuned": True, "truncate": True,
     "attention_factor": None},
    {"type": "linear", "factor": 4.0, "original_max_position_embeddings": 4096, "partial_rotary_factor": 0.5}])
def test_rope_scaling_that_says_nothing_more(scaling):
    """Taken: what refuses the call is that the tables are in host memory (or
    that there is no GPU to ask)."""
    cos = torch.zeros(16, 32)
    with pytest.raises(_lib.EcError):
        ops.rope_table(cos, cos, 1e4, scaling, stream=0)


def test_write_of_more_sequences_than_the_search_counts():
    rc, h = open_()
    assert rc == 0
    for nseq in (-1, (1 << 30) + 1, (1 << 31) - 1):
        refused(L().ec_kv_write(h, 0, 1 << 20, 256, 64, 1 << 20, 256, 64, 4, None, None, nseq, None), "count")
    refused(L().ec_kv_write(h, 0, 1 << 20, 256, 64, 1 << 20, 256, 64, 4, None, None, 1 << 30, None), "cu is NULL")
    assert L().ec_kv_close(h) == 0


def test_handles_until_memory_is_out():
    """A host allocation that fails is an error code; the process goes on."""
    code = ("import sys, os, resource, ctypes as C; sys.path[:0] = [%r, os.path.join(%r, 'lisp-embed_b200'), %r];"
            "from test_ops import L, FAKE; from embedcuda import _lib\n"
            "l, h = L(), C.c_int()\n"
            "size = l.ec_kv_work_size(10, 3)\n"
            "used = int(open('/proc/self/statm').read().split()[0]) * os.sysconf('SC_PAGE_SIZE')\n"
            "resource.setrlimit(resource.RLIMIT_AS, (used + (20 << 20), resource.RLIM_INFINITY))\n"
            "rc, n, ref = 0, 0, C.byref(h)\n"
            "while rc == 0 and n < 4000000:\n"
            "    rc = l.ec_kv_open(FAKE, FAKE, 1, 2, 10, 16, 4, 64, FAKE, 3, 5, FAKE, FAKE, FAKE, size, ref); n += 1\n"
            "resource.setrlimit(resource.RLIMIT_AS, (resource.RLIM_INFINITY, resource.RLIM_INFINITY))\n"
            "assert l.ec_kv_close(h) == 0\n"
            "print(rc, n > 1000, flush=True)\n") % (REPO, REPO, os.path.join(REPO, "tests"))
    out = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=600)
    assert out.returncode == 0, (out.returncode, out.stderr[-500:])
    assert out.stdout.split() == [str(_lib.EC_ENOMEM), "True"]
