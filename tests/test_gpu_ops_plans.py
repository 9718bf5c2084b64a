"""The attention operators over their ways of cutting the work: pairs of
tiles, halves of blocks left out, few and many sequences, few rows, cut
tiles; shared workspaces, strides of single tokens and heads.  References and
tolerances are those of test_gpu_ops.py."""
import random

import pytest
import torch

from test_gpu_ops import (BF16, F16, F32, Cache, attention_reference, check_cached, check_prompt, close, guarded,  # noqa: F401
                          i32, no_wait_gave_up, offsets, ops, rnd)

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------ prompts --
@pytest.mark.parametrize("dt", [BF16, F16])
@pytest.mark.parametrize("lens,hq,hk,hd", [
    ([700] * 40, 8, 4, 128),                # halves, sequences found by bisection
    ([1100] * 34, 2, 2, 64),                # whole blocks, bisection
    ([1300, 5, 0, 1100, 64, 65], 16, 16, 128),  # by tile set
    ([2100, 1900], 14, 2, 128),             # seven heads: tiles of 18 tokens
    ([40, 300, 129, 1] * 30, 10, 5, 96),
])
def test_pairs_of_tiles(ops, dt, lens, hq, hk, hd):
    check_prompt(ops, lens, hq, hk, hd, dt, seed=len(lens), packed=True)


@pytest.mark.parametrize("hq,hk,hd", [(16, 8, 128), (4, 4, 64), (21, 3, 40), (24, 8, 128)])
def test_many_ragged_prompts(ops, hq, hk, hd):
    r = random.Random(hd)
    lens = [r.choice([0, 1, 31, 63, 64, 65, 127, 128, 129, 191, 193, 320]) for _ in range(150)]
    check_prompt(ops, lens, hq, hk, hd, BF16, seed=hq, packed=hd != 40)


@pytest.mark.parametrize("hq,hk", [(128, 1), (100, 1), (65, 1), (256, 2)])
def test_many_heads_to_a_key_head(ops, hq, hk):
    """One token fills a tile, or all but."""
    check_prompt(ops, [1, 70, 0, 300], hq, hk, 64, BF16, seed=hq)
    check_cached(ops, [1, 1, 3], [500, 0, 131], 16, hq, hk, 64, F16, seed=hq)


# -------------------------------------------------------------------- cache --
@pytest.mark.parametrize("dt", [BF16, F16])
@pytest.mark.parametrize("group", [1, 3, 4, 5, 8, 13, 16, 17, 32, 33])
@pytest.mark.parametrize("hd", [64, 128])
def test_rows_of_single_tokens(ops, dt, group, hd):
    """4, 8, 16, 32 rows a tile and more, whole and cut over many CTAs."""
    check_cached(ops, [1, 1, 1, 0], [6000, 17, 900, 50], 32, group, 1, hd, dt, seed=group)


@pytest.mark.parametrize("new", [2, 3, 7, 8, 15, 16])
def test_rows_of_several_tokens(ops, new):
    check_cached(ops, [new, 1, new], [3000, 40, new], 16, 4, 2, 128, BF16, seed=new)


def test_texts_in_pairs_of_tiles(ops):
    """Enough new tokens that nothing is cut, by tile set and by bisection."""
    check_cached(ops, [300, 17, 128, 1] * 6, [700, 17, 900, 333] * 6, 32, 16, 8, 128, BF16, seed=1)
    check_cached(ops, [90, 200, 0] * 14, [500, 200, 40] * 14, 16, 8, 8, 64, F16, seed=2)


def test_one_workspace_for_all(ops):
    """Calls of every kind one after the other in one workspace leave it ready
    for the next: the same bits as from workspaces of their own."""
    c = Cache(ops, [5000, 70, 1200, 9], 16, 2, 128, BF16, seed=6)
    calls = []
    for new, hq in (([1, 1, 1, 1], 4), ([1, 1, 1, 1], 16), ([30, 1, 5, 9], 4), ([1, 0, 0, 0], 64), ([900, 60, 0, 9], 8),
                    ([2, 2, 2, 2], 2), ([1, 1, 1, 1], 4)):
        cu = offsets(new)
        q = rnd(cu[-1], hq, 128, dt=BF16, seed=hq + sum(new))
        calls.append((q, cu, *c.attend(q, cu)))
    size = max(c.h.attention_workspace(q, i32(cu), max(b - a for a, b in zip(cu, cu[1:]))) for q, cu, _, _ in calls)
    work = torch.zeros(size, dtype=torch.uint8, device="cuda")
    for _ in range(3):
        for q, cu, want, lse in calls:
            out, z = c.attend(q, cu, work=work)
            assert torch.equal(out, want) and torch.equal(z, lse)


def test_graphs_that_share_a_workspace(ops):
    """Two captured graphs over one workspace, replayed in turn on one stream."""
    c = Cache(ops, [5000, 70, 1200, 9], 16, 2, 128, BF16, seed=3)
    shapes = [([1, 1, 1, 1], 16), ([40, 20, 7, 9], 8)]
    qs = [rnd(sum(new), hq, 128, dt=BF16, seed=hq) for new, hq in shapes]
    cus = [i32(offsets(new)) for new, _ in shapes]
    want = [c.attend(q, offsets(new))[0] for q, (new, _) in zip(qs, shapes)]
    work = torch.zeros(max(c.h.attention_workspace(q, cu, max(new)) for q, cu, (new, _) in zip(qs, cus, shapes)),
                       dtype=torch.uint8, device="cuda")
    outs, graphs = [torch.zeros_like(q) for q in qs], []
    for q, cu, out, (new, _) in zip(qs, cus, outs, shapes):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            c.h.attention(0, q, cu, out, max(new), work)
        graphs.append(g)
    for turn in (0, 1, 1, 0, 0, 1):
        outs[turn].zero_()
        graphs[turn].replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[turn], want[turn])


# ------------------------------------------------------------------ strides --
def test_strides_of_single_tokens_and_heads(ops):
    """The stride of a dimension of one does not count, whatever it is."""
    q, k, v = rnd(1, 4, 64, dt=BF16, seed=1), rnd(1, 2, 64, dt=BF16, seed=2), rnd(1, 2, 64, dt=BF16, seed=3)
    want = torch.empty_like(q)
    ops.attn_prompt(q, k, v, i32([0, 1]), want)
    odd = [t.as_strided(t.shape, (s, 64, 1)) for t, s in ((q, 3), (k, 1), (v, 0))]
    out = torch.empty_like(q)
    ops.attn_prompt(*odd, i32([0, 1]), out.as_strided(out.shape, (5, 64, 1)))
    assert torch.equal(out, want)
    q, k, v = (rnd(50, 1, 64, dt=F16, seed=i) for i in (4, 5, 6))
    want, out = torch.empty_like(q), torch.empty_like(q)
    ops.attn_prompt(q, k, v, i32([0, 50]), want)
    ops.attn_prompt(*(t.as_strided(t.shape, (64, s, 1)) for t, s in ((q, 7), (k, 0), (v, 1))), i32([0, 50]),
                    out.as_strided(out.shape, (64, 3, 1)))
    assert torch.equal(out, want)
    cos, sin = torch.empty(60, 32, device="cuda"), torch.empty(60, 32, device="cuda")
    ops.rope_table(cos, sin, 1e4)
    a, b = q.clone(), q.clone()
    ops.rope(a, i32(list(range(50))), cos, sin)
    ops.rope(b.as_strided(b.shape, (64, 1, 1)), i32(list(range(50))), cos, sin)
    assert torch.equal(a, b)
    c = Cache(ops, [1], 16, 1, 64, F16)
    c.h.write(0, k[:1].as_strided((1, 1, 64), (3, 1, 1)), v[:1].as_strided((1, 1, 64), (0, 5, 1)), i32([0, 1]))
    got_k, got_v = c.rows(0)
    assert torch.equal(got_k, k[:1]) and torch.equal(got_v, v[:1])


@pytest.mark.parametrize("n", [33, 129, 2500, 4096, 4097, 9000])
def test_lists_of_many_sequences(ops, n):
    """Counted in groups up to 4096 sequences, found by their offsets above;
    runs of empty ones, and a first and last one that is empty."""
    r = random.Random(n)
    lens = [0 if i % 7 < 3 or i in (0, n - 1) else r.choice([1, 5, 40]) for i in range(n)]
    lens[n // 2], lens[n // 3] = 700, 300
    hq, hk, hd = 6, 3, 64
    cu = offsets(lens)
    t = cu[-1]
    q, k, v = rnd(t, hq, hd, dt=BF16, seed=1), rnd(t, hk, hd, dt=BF16, seed=2), rnd(t, hk, hd, dt=BF16, seed=3)
    out, intact = guarded(t, hq, hd, dt=BF16)
    ops.attn_prompt(q, k, v, i32(cu), out)
    intact()
    # all rows were written; some sequences against the reference
    assert not bool((out == 7).all(-1).any())
    some = [n // 2, n // 3] + [i for i in range(n) if lens[i]][:: max(1, n // 40)]
    for i in some:
        a, b = cu[i], cu[i + 1]
        see = torch.ones(b - a, b - a, dtype=torch.bool, device="cuda").tril()
        o, _, tol, _ = attention_reference(q[a:b], k[a:b], v[a:b], see, 1 / 8)
        close(out[a:b], o, tol)
