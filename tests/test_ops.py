"""Refusals of the operators on device buffers: every argument that the host
can see is checked before anything is launched or dereferenced, so none of
these calls needs a GPU (the pointers are never followed)."""
import ctypes as C

import pytest
import torch

from embedcuda import _lib, ops

FAKE = 1 << 20  # 16-byte aligned, never dereferenced
EINVAL = _lib.EC_EINVAL


def L():
    return _lib.lib()


def refused(rc, text):
    assert rc == EINVAL, rc
    assert text in _lib.last_error(), _lib.last_error()


def rope(x=FAKE, xt=256, xh=64, y=2 * FAKE, yt=256, yh=64, dtype=_lib.EC_BF16, tokens=4, heads=4, hd=64, rot=64,
         pos=FAKE, cos=FAKE, sin=FAKE, positions=10):
    return L().ec_rope(x, xt, xh, y, yt, yh, dtype, tokens, heads, hd, rot, 0, 0, pos, cos, sin, positions, None)


def test_rope_refusals():
    refused(rope(dtype=7), "dtype")
    refused(rope(tokens=-1), "rope shape")
    refused(rope(heads=0), "rope shape")
    refused(rope(rot=63), "rot_dim")
    refused(rope(rot=66), "rot_dim")
    refused(rope(rot=0), "rot_dim")
    refused(rope(positions=0), "positions")
    refused(rope(x=None), "NULL")
    refused(rope(pos=None), "NULL")
    refused(rope(x=FAKE + 1), "aligned")
    refused(rope(cos=FAKE + 2), "aligned")
    refused(rope(xh=32), "overlap")
    refused(rope(yt=8), "overlap")
    refused(rope(y=FAKE, yt=512), "in place")
    assert rope(tokens=0, x=None, y=None, pos=None) == 0


def table(positions=8, rot=64, theta=1e4, kind=0, factor=1.0, p0=0.0, p1=0.0, original=0.0, amp=0.0, cos=FAKE):
    return L().ec_rope_table(cos, FAKE, positions, rot, theta, kind, factor, p0, p1, original, amp, None)


def test_rope_table_refusals():
    refused(table(positions=-1), "positions")
    refused(table(rot=3), "rot_dim")
    refused(table(theta=1.0), "theta")
    refused(table(theta=float("nan")), "theta")
    refused(table(kind=4), "scaling")
    refused(table(kind=1, factor=0.5), "factor")
    refused(table(kind=2, factor=8.0, p0=4.0, p1=1.0, original=8192.0), "llama3")
    refused(table(kind=3, factor=8.0, p0=1.0, p1=32.0, original=8192.0), "yarn")
    refused(table(kind=3, factor=8.0, p0=32.0, p1=1.0, original=0.0), "yarn")
    refused(table(amp=-1.0), "amplitude")
    refused(table(cos=None), "NULL")
    assert table(positions=0, cos=None) == 0


def prompt(q=FAKE, qt=512, qh=64, k=FAKE, kt=256, kh=64, out=FAKE, lse=None, dtype=_lib.EC_BF16, tokens=8, hq=8, hk=4,
           hd=64, cu=FAKE, nseq=1, scale=0.0):
    return L().ec_attn_prompt(q, qt, qh, k, kt, kh, k, kt, kh, out, qt, qh, lse, dtype, tokens, hq, hk, hd, cu, nseq,
                              scale, None)


def test_prompt_refusals():
    refused(prompt(dtype=_lib.EC_F32), "bf16 or f16")
    refused(prompt(tokens=-1), "count")
    refused(prompt(tokens=1 << 31), "count")
    refused(prompt(nseq=-1), "count")
    refused(prompt(hd=136, qh=136, kh=136, qt=2048, kt=1024), "head_dim")
    refused(prompt(hd=60), "head_dim")
    refused(prompt(hq=6), "query heads")
    refused(prompt(hk=0), "query heads")
    refused(prompt(scale=-1.0), "scale")
    refused(prompt(scale=float("inf")), "scale")
    refused(prompt(q=None), "NULL")
    refused(prompt(k=None), "NULL")
    refused(prompt(cu=None), "NULL")
    refused(prompt(q=FAKE + 2), "16-byte")
    refused(prompt(qt=516), "multiples of 8")
    refused(prompt(kh=32), "overlap")
    refused(prompt(lse=FAKE + 1), "4-byte")
    assert prompt(tokens=0, q=None, k=None, out=None, cu=None) == 0
    assert prompt(nseq=0) == 0


def open_(k=FAKE, dtype=_lib.EC_BF16, layers=2, pages=10, page=16, heads=4, hd=64, slots=3, width=5, work=FAKE,
          size=None):
    h = C.c_int()
    size = L().ec_kv_work_size(pages, slots) if size is None else size
    return L().ec_kv_open(k, FAKE, dtype, layers, pages, page, heads, hd, FAKE, slots, width, FAKE, FAKE, work,
                          size, C.byref(h)), h.value


def test_cache_refusals():
    refused(open_(k=None)[0], "NULL")
    refused(open_(dtype=_lib.EC_F32)[0], "bf16 or f16")
    refused(open_(layers=0)[0], "cache shape")
    refused(open_(pages=(1 << 20) + 1)[0], "cache shape")
    refused(open_(page=48)[0], "page_size")
    refused(open_(hd=132)[0], "head_dim")
    refused(open_(width=1 << 24, page=128)[0], "2^30")
    refused(open_(layers=65536, pages=1 << 20)[0], "2^30")
    refused(open_(k=FAKE + 8)[0], "16-byte")
    refused(open_(size=16)[0], "work holds")
    refused(L().ec_kv_close(0), "unknown cache handle")
    rc, h = open_()
    assert rc == 0 and h > 0
    try:
        refused(L().ec_kv_reserve(h, FAKE, FAKE, -1, FAKE, None), "negative")
        refused(L().ec_kv_reserve(h, None, FAKE, 1, FAKE, None), "NULL")
        refused(L().ec_kv_fork(h, FAKE, FAKE, 1, None, None), "NULL")
        refused(L().ec_kv_free(h, FAKE + 2, 1, FAKE, None), "4-byte")
        refused(L().ec_kv_compact(h, None, None), "NULL")
        w = lambda layer=0, kt=256, tokens=4, cu=FAKE: L().ec_kv_write(  # noqa: E731
            h, layer, FAKE, kt, 64, FAKE, 256, 64, tokens, cu, None, 1, None)
        refused(w(layer=2), "layer")
        refused(w(kt=32), "overlap")
        refused(w(tokens=-1), "count")
        refused(w(cu=None), "NULL")
        assert w(tokens=0) == 0
        need = L().ec_attn_cached_work_size(h, 4, 8, 1, 4)
        assert need > 0

        def att(layer=0, hq=8, nseq=1, max_new=4, work=FAKE, size=need, tokens=4, cu=FAKE):
            return L().ec_attn_cached(h, layer, FAKE, 512, 64, FAKE, 512, 64, None, tokens, hq, cu, None, nseq,
                                      max_new, 0.0, work, size, None)
        refused(att(layer=-1), "layer")
        refused(att(hq=6), "query heads")
        refused(att(max_new=-1), "max_new")
        refused(att(work=None), "work")
        refused(att(size=need - 1), "work")
        refused(att(nseq=4, size=1 << 30), "slots")
        refused(att(cu=None), "NULL")
        assert att(tokens=0) == 0
    finally:
        assert L().ec_kv_close(h) == 0
    refused(L().ec_kv_compact(h, FAKE, None), "unknown cache handle")


def test_python_layer_refusals():
    """Shapes, types and layouts are checked on the tensors themselves."""
    x = torch.zeros(4, 3, 64, dtype=torch.bfloat16)
    pos = torch.zeros(4, dtype=torch.int32)
    cos = torch.zeros(16, 32)
    with pytest.raises(ValueError, match="dtype"):
        ops.rope(x.double(), pos, cos, cos)
    with pytest.raises(ValueError, match="pos has"):
        ops.rope(x, pos[:3], cos, cos, stream=0)
    with pytest.raises(ValueError, match="int32"):
        ops.rope(x, pos.long(), cos, cos, stream=0)
    with pytest.raises(ValueError, match="adjacent"):
        ops.rope(x.transpose(1, 2), pos, cos, cos, stream=0)
    with pytest.raises(ValueError, match="does not match"):
        ops.rope(x, pos, cos, cos, out=x.float(), stream=0)
    with pytest.raises(ValueError, match="differ"):
        ops.rope(x, pos, cos, cos[:4], stream=0)
    with pytest.raises(ValueError, match="rope_scaling"):
        ops.rope_table(cos, cos, 1e4, {"rope_type": "longrope"}, stream=0)
    cu = torch.tensor([0, 4], dtype=torch.int32)
    kv = torch.zeros(4, 1, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="tokens"):
        ops.attn_prompt(x, kv[:3], kv, cu, x, stream=0)
    with pytest.raises(ValueError, match="k is"):
        ops.attn_prompt(x, kv.half(), kv, cu, x, stream=0)
    with pytest.raises(ValueError, match="expected"):
        ops.attn_prompt(x, kv[..., :32], kv, cu, x, stream=0)
    with pytest.raises(ValueError, match="lse"):
        ops.attn_prompt(x, kv, kv, cu, x, lse=torch.zeros(3, 4), stream=0)
    pool = torch.zeros(1, 4, 16, 1, 64, dtype=torch.bfloat16)
    tab = torch.zeros(2, 3, dtype=torch.int32)
    two, four = torch.zeros(2, dtype=torch.int32), torch.zeros(4, dtype=torch.int32)
    with pytest.raises(ValueError, match="contiguous"):
        ops.KvCache(pool, pool[:, :2], tab, two, four)
    with pytest.raises(ValueError, match="lens"):
        ops.KvCache(pool, pool, tab, four, four)
    with pytest.raises(_lib.EcError, match="page_size"):
        ops.KvCache(pool.view(1, 8, 8, 1, 64), pool.view(1, 8, 8, 1, 64), tab, two, torch.zeros(8, dtype=torch.int32))
    cache = ops.KvCache(pool, pool, tab, two, four)
    with pytest.raises(ValueError, match="status"):
        cache.compact(four, stream=0)
    with pytest.raises(ValueError, match="slots"):
        cache.write(0, kv, kv, torch.zeros(4, dtype=torch.int32), stream=0)
    cache.close()
    with pytest.raises(_lib.EcError, match="unknown cache handle"):
        cache.compact(two, stream=0)


def test_rows_that_are_written_must_not_overlap():
    """A token stride that does not step over a token's heads (nor a head
    stride over the head's tokens) would have two rows in one place."""
    refused(rope(yt=128, yh=64), "overlap")
    refused(prompt(qt=256, qh=64), "overlap")
    refused(prompt(qt=64, qh=256), "overlap")
    # the stride of a single token or head does not count: not refused for it
    assert rope(tokens=0, heads=1, xh=3, yh=5) == 0
    assert prompt(tokens=0, qt=3, kt=5) == 0
