"""Calls at the edges of what the operators on device buffers accept.
References and tolerances are those of test_gpu_ops.py."""
import math
import random

import pytest
import torch

from test_gpu_ops import (BF16, F16, F32, Cache, attention_reference, close, guarded, half_step, i32,  # noqa: F401
                          no_wait_gave_up, offsets, ops, rnd, rope_reference)

pytestmark = pytest.mark.gpu


# -------------------------------------------------------- rotary positions --
@pytest.mark.parametrize("dt", [BF16, F16, F32])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("shift", [1, 2, 4, 8, 12])
def test_rope_tables_at_any_float(ops, dt, interleaved, shift):
    """Tables that start `shift` floats behind a 32-byte boundary (4 and 12: at
    an odd multiple of 16 bytes)."""
    tokens, heads, hd, positions = 70, 5, 128, 40
    n = positions * hd // 2
    cos, sin = (torch.zeros(n + 16, device="cuda")[shift:shift + n].view(positions, hd // 2) for _ in range(2))
    assert cos.data_ptr() % 32 == 4 * shift % 32
    ops.rope_table(cos, sin, 1e4)
    x, pos = rnd(tokens, heads, hd, dt=dt, seed=shift), i32([i % positions for i in range(tokens)])
    out, intact = guarded(tokens, heads, hd, dt=dt)
    ops.rope(x, pos, cos, sin, out=out, interleaved=interleaved)
    ref, tol = rope_reference(x, pos, cos, sin, interleaved, False)
    assert bool(((out.double() - ref).abs() <= tol + half_step(dt) * ref.abs() * 1.01 + torch.finfo(dt).tiny).all())
    intact()


# --------------------------------------------------------------------- pages --
@pytest.mark.parametrize("slots,n", [(3, 4), (3, 5000), (1, 70000), (40, 41), (2000, 2001)])
def test_lists_longer_than_the_cache_has_slots(ops, slots, n):
    """They name a slot twice, whatever they hold: refused, nothing changed,
    and what lies behind the caller's scratch is not looked at."""
    lens = [20, 5, 0][:slots]
    c = Cache(ops, lens, 16, 1, 16, F16, spare=4, seed=1, width=6, slots=slots)
    before = c.state()
    src, dst = i32([i % slots for i in range(n)]), i32([(i + 1) % slots for i in range(n)])
    calls = (lambda: c.h.reserve(src, i32([1] * n), c.status), lambda: c.h.fork(src, dst, c.status),
             lambda: c.h.fork(i32([0] * n), i32([slots - 1] * n), c.status), lambda: c.h.free(src, c.status))
    for call in calls:
        c.status.fill_(9)
        call()
        assert c.status.tolist() == [2, 0]
        for a, b in zip(c.state(), before):
            assert torch.equal(a, b)
    if slots > 2:  # and the cache goes on as before
        c.h.fork(i32([0]), i32([2]), c.status)
        assert c.status.tolist() == [0, 1] and c.lens.tolist()[:3] == [20, 5, 20]


# ----------------------------------------------------------- cached attention --
@pytest.mark.parametrize("keys,sequences", [(4_193_920 - 128, 148), (4_193_920, 148), (4_200_005, 148), (8_400_001, 74)])
def test_a_tile_for_every_cta_behind_millions_of_keys(ops, keys, sequences):
    """The last key takes all the weight: the others' scores are 56 below it,
    4e6 e^-56 < 2^-56.  Left out, the result would be the others' mean."""
    page, hd = 128, 8
    pages = -(-keys // page)
    k = torch.zeros(1, pages, page, 1, hd, device="cuda", dtype=BF16)
    v = rnd(1, pages, page, 1, hd, dt=BF16, seed=1)
    at = (0, (keys - 1) // page, (keys - 1) % page)
    k[at][0, 0] = 20.0
    tables = torch.arange(pages, device="cuda", dtype=torch.int32)[None]
    h = ops.KvCache(k, v, tables, i32([keys]), torch.ones(pages, device="cuda", dtype=torch.int32))
    q = torch.zeros(sequences, 1, hd, device="cuda", dtype=BF16)
    q[..., 0] = 8.0
    cu, slots = i32(range(sequences + 1)), i32([0] * sequences)
    work = torch.zeros(h.attention_workspace(q, cu, 1), dtype=torch.uint8, device="cuda")
    for _ in range(2):
        out, intact = guarded(sequences, 1, hd, dt=BF16)
        h.attention(0, q, cu, out, 1, work, slots=slots)
        assert bool((out[:, 0] == v[at][0]).all())
        intact()
    # the workspace is left ready for a call that is cut
    out, intact = guarded(3, 1, hd, dt=BF16)
    h.attention(0, q[:3], cu[:4], out, 1, work, slots=slots[:3])
    assert bool((out[:, 0] == v[at][0]).all())
    intact()


@pytest.mark.parametrize("new", [1, 40])
def test_offsets_that_descend_again_and_again(ops, new):
    """Every other sequence is all the tokens of the call (here 1024 times, with
    more units of work than 32 bits hold): nothing outside the rows is written,
    and the workspace is left ready."""
    t, hk, hd, page, pages = 4096, 8, 8, 128, 512
    k, v = (rnd(1, pages, page, hk, hd, dt=BF16, seed=i) for i in (1, 2))
    tables = torch.arange(pages, device="cuda", dtype=torch.int32)[None]
    h = ops.KvCache(k, v, tables, i32([page * pages]), torch.ones(pages, device="cuda", dtype=torch.int32))
    q = rnd(t, hk, hd, dt=BF16, seed=3)
    cu, slots = i32([0, t] * 1024 + [0]), i32([0] * 2048)
    good = i32([0, 5])
    work = torch.zeros(max(h.attention_workspace(q, cu, new), h.attention_workspace(q[:5], good, 5)), dtype=torch.uint8,
                       device="cuda")
    want, out = (torch.empty_like(q[:5]) for _ in range(2))
    h.attention(0, q[:5], good, want, 5, work.clone(), slots=slots[:1])
    rows, intact = guarded(t, hk, hd, dt=BF16)
    lse, intact_l = guarded(t, hk, dt=F32)
    h.attention(0, q, cu, rows, new, work, slots=slots, lse=lse)
    h.attention(0, q[:5], good, out, 5, work, slots=slots[:1])
    torch.cuda.synchronize()
    intact(), intact_l()
    assert torch.equal(out, want)


@pytest.mark.parametrize("n", [33, 400, 4096, 4097])
def test_prompt_offsets_that_descend_again_and_again(ops, n):
    t, hd = 3000, 64
    q, k, v = (rnd(t, 2, hd, dt=BF16, seed=h) for h in range(3))
    out, intact = guarded(t, 2, hd, dt=BF16)
    lse, intact_l = guarded(t, 2, dt=F32)
    ops.attn_prompt(q, k, v, i32([t * (i & 1) for i in range(n + 1)]), out, lse=lse)
    torch.cuda.synchronize()
    intact(), intact_l()


# -------------------------------------------------------------- where it lies --
@pytest.mark.parametrize("which", range(6))
def test_cache_memory_of_the_host_is_refused(ops, which):
    """Any of the six buffers of a cache, by every call that would launch."""
    import ctypes as C
    from embedcuda import _lib
    L = _lib.lib()
    k, v = (torch.zeros(1, 8, 16, 1, 64, dtype=BF16) for _ in range(2))
    tables, lens, refs = torch.zeros(2, 3, dtype=torch.int32), i32([0, 0]).cpu(), torch.zeros(8, dtype=torch.int32)
    work = torch.zeros(L.ec_kv_work_size(8, 2), dtype=torch.uint8)
    bufs = [t if i == which else t.cuda() for i, t in enumerate((k, v, tables, lens, refs, work))]
    k, v, tables, lens, refs, work = (t.data_ptr() for t in bufs)
    h = C.c_int()
    assert L.ec_kv_open(k, v, _lib.EC_BF16, 1, 8, 16, 1, 64, tables, 2, 3, lens, refs, work, bufs[5].numel(),
                        C.byref(h)) == 0
    one, status, cu = i32([0]), i32([9, 9]), i32([0, 1])
    x = torch.zeros(1, 1, 64, device="cuda", dtype=BF16)
    scratch = torch.zeros(L.ec_attn_cached_work_size(h.value, 1, 1, 1, 1), dtype=torch.uint8, device="cuda")
    st = torch.cuda.current_stream().cuda_stream
    p = lambda t: t.data_ptr()  # noqa: E731
    calls = (lambda: L.ec_kv_reserve(h, p(one), p(one), 1, p(status), st),
             lambda: L.ec_kv_fork(h, p(one), p(one), 1, p(status), st),
             lambda: L.ec_kv_free(h, p(one), 1, p(status), st),
             lambda: L.ec_kv_compact(h, p(status), st),
             lambda: L.ec_kv_write(h, 0, p(x), 64, 64, p(x), 64, 64, 1, p(cu), None, 1, st),
             lambda: L.ec_attn_cached(h, 0, p(x), 64, 64, p(x), 64, 64, None, 1, 1, p(cu), None, 1, 1, 0.0,
                                      p(scratch), scratch.numel(), st))
    for call in calls:
        for _ in range(2):
            assert call() == _lib.EC_EINVAL
            assert "the cache's memory" in _lib.last_error() and "device memory" in _lib.last_error()
    assert status.tolist() == [9, 9]
    assert L.ec_kv_close(h) == 0


def test_cache_lists_of_the_host_are_refused(ops):
    from embedcuda import _lib
    c = Cache(ops, [5, 0], 16, 1, 64, BF16)
    for _ in range(2):  # before and after a call that was right
        with pytest.raises(_lib.EcError, match="device memory"):
            c.h.reserve(i32([0]).cpu(), i32([1]), c.status)
        c.h.reserve(i32([0]), i32([1]), c.status)
        assert c.status.tolist() == [0, 0]
    with pytest.raises(ValueError, match="tables is on cpu"):
        ops.KvCache(c.k, c.v, c.tables.cpu(), c.lens, c.refs)


def test_compaction_past_32_bits(ops):
    """The r-th page in use at or above their number goes to the r-th hole below
    it: 9, 16500, 17000 and 17999 to 0, 1, 2 and 3, contents and table."""
    layers, pages, page, hk, hd = 2, 18000, 128, 8, 128  # 2.36e9 elements a layer
    k, v = (torch.empty(layers, pages, page, hk, hd, device="cuda", dtype=BF16) for _ in range(2))
    mine = [17999, 16500, 9, 17000]
    for x, s in ((k, 1), (v, 2)):
        x[:, mine] = rnd(layers, 4, page, hk, hd, dt=BF16, seed=s)
    want = [x[:, mine].clone() for x in (k, v)]
    tables, lens, refs = i32([mine + [-1]]), i32([450]), torch.zeros(pages, dtype=torch.int32, device="cuda")
    refs[mine] = 1
    h, status = ops.KvCache(k, v, tables, lens, refs), i32([9, 9])
    h.compact(status)
    assert status.tolist() == [0, 4]
    assert tables.tolist() == [[3, 1, 0, 2, -1]] and lens.tolist() == [450]
    assert refs.nonzero()[:, 0].tolist() == [0, 1, 2, 3] and refs[:4].tolist() == [1] * 4
    for x, w in zip((k, v), want):
        assert torch.equal(x[:, [3, 1, 0, 2]], w)
    h.compact(status)
    assert status.tolist() == [0, 0] and tables.tolist() == [[3, 1, 0, 2, -1]]


# ------------------------------------- infinities and NaN that are not seen --
def _poisoned(t, hk, hd, dt, seed, places):
    """Values [t, hk, hd] with NaN and infinities at (token, head, element)."""
    v = rnd(t, hk, hd, dt=dt, seed=seed)
    for i, (tok, h, e) in enumerate(places):
        v[tok, h, e] = (math.nan, math.inf, -math.inf)[i % 3]
    return v


def _seen(v, see):
    """[m, hk, hd]: what a row gets where it sees a value that is not finite
    (NaN, or an infinity of one sign); 0 where all that it sees is finite."""
    see, v = see[:, :, None, None], v.double()[None]
    nan = (see & v.isnan()).any(1)
    up, down = (see & (v == math.inf)).any(1), (see & (v == -math.inf)).any(1)
    r = torch.zeros_like(nan, dtype=torch.float64)
    r[up], r[down], r[nan | (up & down)] = math.inf, -math.inf, math.nan
    return r


def _check_unseen(out, lse, q, k, v, see, scale):
    """Rows are right wherever they see finite values only; where they see an
    infinity or a NaN they are not finite, as the definition has it."""
    bad = _seen(v, see).repeat_interleave(q.shape[1] // k.shape[1], 1)
    o, z, tol, tol_z = attention_reference(q, k, v.nan_to_num(0, 0, 0), see, scale)
    fine = bad == 0
    assert bool(fine.any()) and not bool(fine.all())
    close(out[fine], o[fine], tol[fine])
    assert not bool(out[~fine].isfinite().any())
    close(lse, z, tol_z)


@pytest.mark.parametrize("dt", [BF16, F16])
@pytest.mark.parametrize("hq,hk,hd", [(16, 8, 128), (4, 1, 64), (6, 2, 96), (14, 2, 128), (2, 2, 8), (128, 1, 64)])
@pytest.mark.parametrize("lens", [[300], [90, 40, 257], [200] * 40])
def test_prompt_values_that_are_not_seen(ops, dt, hq, hk, hd, lens):
    r = random.Random(hq + len(lens))
    cu = offsets(lens)
    places = []
    for a, b in zip(cu, cu[1:]):
        places += [(r.randrange(a, b), r.randrange(hk), r.randrange(hd)) for _ in range(r.choice([1, 2]))]
        places.append((b - 1, r.randrange(hk), r.randrange(hd)))
    t = cu[-1]
    q, k = rnd(t, hq, hd, dt=dt, seed=1), rnd(t, hk, hd, dt=dt, seed=2)
    v = _poisoned(t, hk, hd, dt, 3, places)
    out, intact = guarded(t, hq, hd, dt=dt)
    lse, intact_l = guarded(t, hq, dt=F32)
    ops.attn_prompt(q, k, v, i32(cu), out, lse=lse)
    intact(), intact_l()
    for a, b in list(zip(cu, cu[1:]))[:3]:
        see = torch.ones(b - a, b - a, dtype=torch.bool, device="cuda").tril()
        _check_unseen(out[a:b], lse[a:b], q[a:b], k[a:b], v[a:b], see, hd ** -0.5)


@pytest.mark.parametrize("hq,hk,hd,page", [(8, 2, 128, 32), (4, 4, 64, 16), (6, 2, 96, 128), (3, 1, 40, 64)])
@pytest.mark.parametrize("new,past", [([4], [700]), ([2, 3, 1], [40, 127, 0]), ([16, 5], [3000, 64]), ([200], [5000]),
                                      ([300, 77], [0, 900]), ([60] * 30, [90] * 30), ([2] * 40, [900] * 40)])
def test_cached_values_that_are_not_seen(ops, hq, hk, hd, page, new, past):
    """Few rows, cut tiles and whole ones: a value among the new tokens reaches
    only those behind it."""
    r = random.Random(sum(new) + hq)
    kv = [a + b for a, b in zip(new, past)]
    c = Cache(ops, kv, page, hk, hd, BF16, seed=4, layers=2)
    for s, (n, m) in enumerate(zip(new, kv)):
        for i in range(2):
            tok = m - 1 if i == 0 else r.randrange(m - n, m)
            c.v[1, int(c.tables[s, tok // page]), tok % page, r.randrange(hk), r.randrange(hd)] = (math.nan, math.inf)[i]
    cu = offsets(new)
    q = rnd(cu[-1], hq, hd, dt=BF16, seed=5)
    out, lse = c.attend(q, cu, layer=1)
    for s in range(min(3, len(new))):
        a, b = cu[s], cu[s + 1]
        k, v = c.rows(s, 1)
        pos = torch.arange(b - a, device="cuda")[:, None] + kv[s] - (b - a)
        see = torch.arange(kv[s], device="cuda") <= pos
        if b - a > 1:
            _check_unseen(out[a:b], lse[a:b], q[a:b], k, v, see, hd ** -0.5)


def test_all_values_nan(ops):
    """Nothing to compute again that would be finite, and in no time that the
    waits would notice."""
    for hq, hk, t in ((8, 8, 6000), (4, 1, 3000)):
        q, k = rnd(t, hq, 128, dt=BF16, seed=1), rnd(t, hk, 128, dt=BF16, seed=2)
        v = torch.full((t, hk, 128), math.nan, device="cuda", dtype=BF16)
        out = torch.zeros_like(q)
        ops.attn_prompt(q, k, v, i32([0, t // 2, t]), out)
        assert bool(out.isnan().all())
        v[:, :, 1:] = 0
        ops.attn_prompt(q, k, v, i32([0, t // 2, t]), out)
        assert bool(out[..., 0].isnan().all()) and bool((out[..., 1:] == 0).all())
