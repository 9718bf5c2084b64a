"""The operators on device buffers against their definitions in 64 bits.

Tolerances are derived, element by element, from the roundings that the
kernels are allowed (u = half a unit of the type relative to the value):

* rotary positions: y = x0 c - x1 s in fp32 (three roundings of 2^-24 on
  |x0 c| + |x1 s|), rounded once to the type: u |y|.
* attention: with p the exact probabilities and A = sum_j p_j |v_j|:
  - a probability is rounded to the type for the product with v: u A
    (f16 also loses what lies below its smallest subnormal: 2^-25 a key,
    times max |v|); the denominator sums unrounded probabilities;
  - a score is an fp32 sum of head_dim products and is scaled: its error d is
    at most (head_dim + 4) 2^-24 scale * max_j sum_i |q_i k_ji|, and the
    exponential adds 2^-21 relative; numerator and denominator move by
    exp(d) each: 2 (d + 2^-21) A;
  - the product with v is an fp32 sum over the keys: keys * 2^-24 A;
  - the result is rounded to the type: u |o|.
* log-sum-exp: d + 2^-21 + keys * 2^-24, and 2^-23 of its own size.
"""
import math
import random

import pytest
import torch

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def half_step(dt):
    return torch.finfo(dt).eps / 2


@pytest.fixture(scope="module")
def ops(ec):
    from embedcuda import ops
    return ops


@pytest.fixture(scope="module", autouse=True)
def no_wait_gave_up(ec):
    """Every kernel's bounded waits ended by themselves."""
    yield
    torch.cuda.synchronize()
    assert ec.lib().ec_op_status() == 0, ec.last_error()


def rnd(*shape, dt=F32, seed=0, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, device="cuda", generator=g) * scale).to(dt)


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def offsets(lens):
    cu = [0]
    for n in lens:
        cu.append(cu[-1] + n)
    return cu


def guarded(*shape, dt, fill=7.0):
    """A tensor inside a larger one of a known value, and a check that what
    lies around it kept that value."""
    n = math.prod(shape)
    whole = torch.full((n + 512,), fill, device="cuda", dtype=dt)
    part = whole[256:256 + n].view(*shape)

    def intact():
        assert bool((whole[:256] == fill).all()) and bool((whole[256 + n:] == fill).all())
    return part, intact


# -------------------------------------------------------- rotary positions --
def rope_reference(x, pos, cos, sin, interleaved, inverse):
    """64 bits; also the bound of the fp32 arithmetic before the last rounding."""
    half = cos.shape[1]
    x = x.double()
    c, s = cos[pos.long()].double()[:, None], sin[pos.long()].double()[:, None]
    s = -s if inverse else s
    i0 = torch.arange(half, device="cuda") * (2 if interleaved else 1)
    i1 = i0 + (1 if interleaved else half)
    a, b = x[..., i0], x[..., i1]
    y, e = x.clone(), torch.zeros_like(x)
    y[..., i0], y[..., i1] = a * c - b * s, b * c + a * s
    e[..., i0], e[..., i1] = (a * c).abs() + (b * s).abs(), (b * c).abs() + (a * s).abs()
    return y, 3 * 2.0 ** -24 * e


@pytest.mark.parametrize("dt", [BF16, F16, F32])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("tokens,heads,hd,rot,inverse", [
    (1, 24, 128, 128, False), (1, 1, 2, 2, False), (37, 3, 80, 80, True), (300, 5, 96, 40, False),
    (1023, 8, 64, 64, True), (6, 7, 36, 18, False), (2049, 2, 256, 128, False), (5, 9, 130, 130, True)])
def test_rope(ops, dt, interleaved, tokens, heads, hd, rot, inverse):
    g = random.Random(tokens + hd)
    x = rnd(tokens, heads + 2, hd, dt=dt, seed=tokens)[:, 1:heads + 1]
    cos, sin = rnd(50, rot // 2, seed=1), rnd(50, rot // 2, seed=2)
    pos = i32([g.randrange(50) for _ in range(tokens)])
    out, intact = guarded(tokens, heads, hd, dt=dt)
    keep = x.clone()
    ops.rope(x, pos, cos, sin, out=out, interleaved=interleaved, inverse=inverse)
    ref, tol = rope_reference(x, pos, cos, sin, interleaved, inverse)
    tol = tol + half_step(dt) * ref.abs() * 1.01 + torch.finfo(dt).tiny
    assert bool(((out.double() - ref).abs() <= tol).all())
    assert torch.equal(x, keep)
    intact()
    # in place, the same bits; the heads around are left alone
    wide = rnd(tokens, heads + 2, hd, dt=dt, seed=tokens)
    before = wide.clone()
    ops.rope(wide[:, 1:heads + 1], pos, cos, sin, interleaved=interleaved, inverse=inverse)
    assert torch.equal(wide[:, 1:heads + 1], out)
    assert torch.equal(wide[:, 0], before[:, 0]) and torch.equal(wide[:, -1], before[:, -1])


def test_rope_layouts_positions_and_gradient(ops):
    """Heads first, odd bases, positions that are none or past the table, and
    the inverse as the gradient (against differences and by turning back)."""
    cos, sin = torch.empty(64, 16, device="cuda"), torch.empty(64, 16, device="cuda")
    ops.rope_table(cos, sin, 1e4)
    x = rnd(5, 40, 32, dt=F32, seed=3).transpose(0, 1)  # [40 tokens, 5 heads, 32]
    pos = i32([i % 64 for i in range(40)])
    y = ops.rope(x, pos, cos, sin, out=torch.empty(40, 5, 32, device="cuda"))
    ref, tol = rope_reference(x, pos, cos, sin, False, False)
    assert bool(((y.double() - ref).abs() <= tol + 2.0 ** -24 * ref.abs()).all())
    # a base that only elements are aligned to
    odd = rnd(1 + 40 * 5 * 32, dt=BF16, seed=4)[1:].view(40, 5, 32)
    got = ops.rope(odd, pos, cos, sin, out=torch.empty_like(odd))
    ref, tol = rope_reference(odd, pos, cos, sin, False, False)
    assert bool(((got.double() - ref).abs() <= tol + 2.0 ** -8 * 1.01 * ref.abs()).all())
    # positions: -1 leaves the row, 64 and INT32_MAX are past the table
    pos2 = pos.clone()
    pos2[3], pos2[7], pos2[9] = -1, 64, 2 ** 31 - 1
    out = torch.full((40, 5, 32), 5.0, device="cuda")
    ops.rope(x, pos2, cos, sin, out=out)
    assert bool((out[3] == 5.0).all()) and bool(out[[7, 9]].isnan().all())
    rest = [i for i in range(40) if i not in (3, 7, 9)]
    assert torch.equal(out[rest], y[rest])
    # the gradient of sum(w * rope(x)) is the inverse turn of w; it is linear
    # in x, so a difference over any step gives it exactly but for rounding
    w = rnd(40, 5, 32, seed=6)
    grad = ops.rope(w, pos, cos, sin, out=torch.empty_like(w), inverse=True)
    d = rnd(40, 5, 32, seed=7)
    up = ops.rope((x + d).contiguous(), pos, cos, sin, out=torch.empty_like(w))
    down = ops.rope((x - d).contiguous(), pos, cos, sin, out=torch.empty_like(w))
    diff = ((up.double() - down.double()) / 2 * w.double()).sum()
    want = (grad.double() * d.double()).sum()
    # 6400 terms of size ~1, each with a few roundings of values up to ~8
    assert abs(float(diff - want)) <= 6400 * 8 * 8 * 2.0 ** -24
    back = ops.rope(y, pos, cos, sin, out=torch.empty_like(w), inverse=True)
    assert bool(((back - x).abs() <= 8 * 2.0 ** -24 * 8).all())


@pytest.mark.parametrize("scaling", [
    None, {"rope_type": "linear", "factor": 3.0},
    {"rope_type": "llama3", "factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0,
     "original_max_position_embeddings": 8192},
    {"type": "yarn", "factor": 4.0, "original_max_position_embeddings": 4096},
    {"rope_type": "yarn", "factor": 16.0, "beta_fast": 16.0, "beta_slow": 2.0, "attention_factor": 1.25,
     "original_max_position_embeddings": 2048}])
@pytest.mark.parametrize("positions,rot,theta", [(1, 2, 1e4), (1000, 64, 1e4), (70001, 128, 1e6), (33, 40, 5e5)])
def test_rope_table(ops, scaling, positions, rot, theta):
    cos, intact_c = guarded(positions, rot // 2, dt=F32)
    sin, intact_s = guarded(positions, rot // 2, dt=F32)
    ops.rope_table(cos, sin, theta, scaling)
    s = scaling or {}
    kind = s.get("rope_type", s.get("type"))
    f, amp = [], 1.0
    for i in range(rot // 2):
        w = theta ** (-2.0 * i / rot)
        if kind == "linear":
            w /= s["factor"]
        if kind == "llama3":
            wave = 2 * math.pi / w
            if wave > 8192:
                w /= 8.0
            elif wave >= 2048:
                r = (8192 / wave - 1.0) / 3.0
                w = (1 - r) * w / 8.0 + r * w
        if kind == "yarn":
            n = s["original_max_position_embeddings"]
            at = lambda b: rot * math.log(n / (b * 2 * math.pi)) / (2 * math.log(theta))  # noqa: E731
            lo = max(math.floor(at(s.get("beta_fast", 32.0))), 0)
            hi = min(math.ceil(at(s.get("beta_slow", 1.0))), rot - 1)
            r = min(1.0, max(0.0, (i - lo) / max(hi - lo, 1e-3)))
            w = w / s["factor"] * r + w * (1 - r)
            amp = s.get("attention_factor", 0.1 * math.log(s["factor"]) + 1)
        f.append(w)
    ang = torch.outer(torch.arange(positions, dtype=torch.float64), torch.tensor(f, dtype=torch.float64)).cuda()
    # one rounding to fp32 of values up to amp; angles up to 7e4 in double
    # carry 7e4 * a few 2^-53
    tol = 2.0 ** -24 * amp + 7e4 * 2.0 ** -50
    assert float((cos.double() - ang.cos() * amp).abs().max()) <= tol
    assert float((sin.double() - ang.sin() * amp).abs().max()) <= tol
    intact_c()
    intact_s()


# ---------------------------------------------------------------- attention --
def attention_reference(q, k, v, see, scale):
    """q [m, hq, d], k and v [n, hk, d], see [m, n] -> out, lse and their
    bounds (see the module's text)."""
    m, hq, d = q.shape
    n, hk = k.shape[:2]
    u = half_step(q.dtype)
    dt = q.dtype
    q, k, v = q.double(), k.double(), v.double()
    k, v = (t.repeat_interleave(hq // hk, 1) for t in (k, v))
    s = torch.einsum("mhd,nhd->hmn", q, k) * scale
    size = torch.einsum("mhd,nhd->hmn", q.abs(), k.abs()) * scale
    s = s.masked_fill(~see, -math.inf)
    size = size.masked_fill(~see, 0.0)
    if n == 0:
        z = torch.zeros(m, hq, d, dtype=torch.float64, device=q.device)
        return z, z[..., 0] - math.inf, z, z[..., 0]
    lse = torch.logsumexp(s, -1)
    p = torch.exp(s - torch.where(lse == -math.inf, 0.0, lse)[..., None])
    out = torch.einsum("hmn,nhd->mhd", p, v)
    big = torch.einsum("hmn,nhd->mhd", p, v.abs())
    err = ((d + 4) * 2.0 ** -24 * size.amax(-1) + 2.0 ** -21).T  # [m, hq]
    tol = (u + 2 * err[..., None] + n * 2.0 ** -24) * big + u * 1.01 * out.abs()
    if dt == F16:
        tol = tol + n * 2.0 ** -25 * v.abs().amax(0) + 2.0 ** -25
    lse = lse.T
    return out, lse, tol + 1e-30, err + n * 2.0 ** -24 + 2.0 ** -23 * lse.abs().nan_to_num(posinf=0.0)


def close(got, want, tol):
    assert got.shape == want.shape
    same = (got.double() == want)  # infinities
    bad = ~(same | ((got.double() - want).abs() <= tol))
    assert not bool(bad.any()), (int(bad.sum()), float((got.double() - want).abs()[bad].nan_to_num(99).max()))


def check_prompt(ops, lens, hq, hk, hd, dt, seed=0, packed=False, scale=0.0, behind=3, q_scale=1.0):
    cu = offsets(lens)
    t = cu[-1] + behind
    if packed:
        x = rnd(t, hq + 2 * hk, hd, dt=dt, seed=seed)
        q, k, v = x[:, :hq], x[:, hq:hq + hk], x[:, hq + hk:]
    else:
        q, k, v = (rnd(t, h, hd, dt=dt, seed=seed + i) for i, h in enumerate((hq, hk, hk)))
    q.mul_(q_scale)
    k[cu[-1]:], v[cu[-1]:] = math.nan, math.inf  # behind the last sequence
    out, intact = guarded(t, hq, hd, dt=dt)
    lse, intact_l = guarded(t, hq, dt=F32)
    ops.attn_prompt(q, k, v, i32(cu), out, lse=lse, scale=scale)
    for a, b in zip(cu, cu[1:]):
        if a == b:
            continue
        see = torch.ones(b - a, b - a, dtype=torch.bool, device="cuda").tril()
        o, z, tol, tol_z = attention_reference(q[a:b], k[a:b], v[a:b], see, scale or 1 / math.sqrt(hd))
        close(out[a:b], o, tol)
        close(lse[a:b], z, tol_z)
    assert bool((out[cu[-1]:] == 7).all()) and bool((lse[cu[-1]:] == 7).all())
    intact()
    intact_l()
    return out


SHAPES = [(16, 8, 128), (14, 2, 64), (8, 8, 32), (3, 1, 96), (10, 2, 128), (8, 1, 64), (21, 3, 40), (2, 2, 8),
          (12, 2, 120), (17, 1, 16)]


@pytest.mark.parametrize("dt", [BF16, F16])
@pytest.mark.parametrize("hq,hk,hd", SHAPES)
def test_prompt_shapes(ops, dt, hq, hk, hd):
    check_prompt(ops, [1, 0, 5, 64, 127, 128, 129, 31], hq, hk, hd, dt, seed=hq + hd, packed=hd % 16 == 0)


@pytest.mark.parametrize("lens", [[1], [2], [0, 0, 1, 0], [128], [256], [257], [513, 1], [1] * 40, [1000, 3, 700],
                                  [2500]])
@pytest.mark.parametrize("hq,hk", [(4, 2), (7, 1)])
def test_prompt_lengths(ops, lens, hq, hk):
    check_prompt(ops, lens, hq, hk, 128, BF16, seed=sum(lens), packed=True)


def test_prompt_many_sequences(ops):
    r = random.Random(5)
    check_prompt(ops, [r.choice([0, 1, 3, 17, 130, 260]) for _ in range(150)], 4, 2, 64, F16, seed=9)


def test_prompt_scale_and_large_scores(ops):
    """A scale of one's own, and scores whose maximum moves by hundreds from
    key to key (the running maximum has to follow)."""
    check_prompt(ops, [300, 77], 4, 2, 128, BF16, scale=0.5, seed=1)
    check_prompt(ops, [300, 77], 4, 2, 64, BF16, q_scale=30.0, seed=2)
    check_prompt(ops, [200], 2, 1, 64, F16, scale=1e-3, seed=3)


def test_prompt_rising_and_falling_maximum(ops):
    """Keys whose scores rise, or fall, steadily over 600 positions."""
    n, hd = 600, 64
    for sign in (1.0, -1.0):
        q = torch.zeros(n, 2, hd, device="cuda", dtype=BF16)
        q[..., 0] = 8.0
        k = torch.zeros(n, 1, hd, device="cuda", dtype=BF16)
        k[:, 0, 0] = (sign * torch.arange(n, device="cuda") / 4).to(BF16)
        v = rnd(n, 1, hd, dt=BF16, seed=3)
        out = torch.empty(n, 2, hd, device="cuda", dtype=BF16)
        ops.attn_prompt(q, k, v, i32([0, n]), out)
        see = torch.ones(n, n, dtype=torch.bool, device="cuda").tril()
        o, _, tol, _ = attention_reference(q, k, v, see, 1 / 8)
        close(out, o, tol)


def test_prompt_sequences_do_not_mix(ops):
    """NaN and infinities in one sequence reach no other one, whichever tile
    they share; scores of -infinity leave no weight."""
    cu, hd = [0, 50, 90, 200], 64
    q, k, v = (rnd(200, h, hd, dt=BF16, seed=h) for h in (4, 2, 2))
    out, clean = torch.empty_like(q), torch.empty_like(q)
    ops.attn_prompt(q, k, v, i32(cu), clean)
    k[50:90], v[50:90], q[50:90] = math.nan, math.inf, -math.inf
    ops.attn_prompt(q, k, v, i32(cu), out)
    assert torch.equal(out[:50], clean[:50]) and torch.equal(out[90:], clean[90:])
    assert bool(out[50:90].isnan().all())


def test_prompt_heads_first_and_large_strides(ops):
    t, hq, hk, hd = 190, 6, 2, 64
    q, k, v = (rnd(h, t, hd, dt=F16, seed=h).transpose(0, 1) for h in (hq, hk, hk))
    wide = rnd(t, hq, 3 * hd, dt=F16, seed=1)
    out = wide[..., hd:2 * hd]
    keep = wide.clone()
    ops.attn_prompt(q, k, v, i32([0, 100, t]), out)
    for a, b in ((0, 100), (100, t)):
        see = torch.ones(b - a, b - a, dtype=torch.bool, device="cuda").tril()
        o, _, tol, _ = attention_reference(q[a:b], k[a:b], v[a:b], see, 1 / 8)
        close(out[a:b], o, tol)
    assert torch.equal(wide[..., :hd], keep[..., :hd]) and torch.equal(wide[..., 2 * hd:], keep[..., 2 * hd:])


def test_prompt_bad_offsets_stay_in_range(ops):
    """Offsets that pass the buffers or run backwards write nothing outside
    the rows of the call."""
    t, hd = 100, 64
    q, k, v = (rnd(t, 2, hd, dt=BF16, seed=h) for h in range(3))
    for cu in ([0, 50, 300], [-40, 20, 100], [0, 80, 30, 100], [2 ** 31 - 1, 2 ** 31 - 1], [0, 2 ** 31 - 1]):
        out, intact = guarded(t, 2, hd, dt=BF16)
        lse, intact_l = guarded(t, 2, dt=F32)
        ops.attn_prompt(q, k, v, i32(cu), out, lse=lse)
        torch.cuda.synchronize()
        intact()
        intact_l()


# -------------------------------------------------------------------- cache --
class Cache:
    """A cache whose slots hold `lens` random tokens in pages in no order."""

    def __init__(self, ops, lens, page, hk, hd, dt, layers=1, spare=3, seed=0, width=None, slots=None):
        r = random.Random(seed)
        need = [-(-n // page) for n in lens]
        self.pages = max(1, sum(need) + spare)
        order = list(range(self.pages))
        r.shuffle(order)
        width = width or max([1] + need) + 1
        rows, refs = [], [0] * self.pages
        for n in need:
            mine = [order.pop() for _ in range(n)]
            for p in mine:
                refs[p] = 1
            rows.append(mine + [-1] * (width - n))
        for _ in range((slots or len(lens)) - len(lens)):
            rows.append([-1] * width)
        self.k, self.v = (rnd(layers, self.pages, page, hk, hd, dt=dt, seed=seed + i) for i in (1, 2))
        self.tables, self.refs = i32(rows), i32(refs)
        self.lens = i32(list(lens) + [0] * (len(rows) - len(lens)))
        self.page = page
        self.status = i32([9, 9])
        self.h = ops.KvCache(self.k, self.v, self.tables, self.lens, self.refs)

    def rows(self, slot, layer=0):
        n = int(self.lens[slot])
        p = self.tables[slot, :-(-n // self.page)].long()
        f = lambda x: x[layer][p].reshape(-1, *x.shape[3:])[:n]  # noqa: E731
        return f(self.k), f(self.v)

    def state(self):
        return [x.clone() for x in (self.k, self.v, self.tables, self.lens, self.refs)]

    def attend(self, q, cu, slots=None, layer=0, scale=0.0, max_new=None, work=None):
        out, intact = guarded(*q.shape, dt=q.dtype)
        lse, intact_l = guarded(*q.shape[:2], dt=F32)
        new = max([0] + [b - a for a, b in zip(cu, cu[1:])]) if max_new is None else max_new
        cu = i32(cu)
        if work is None:
            work = torch.zeros(self.h.attention_workspace(q, cu, new), dtype=torch.uint8, device="cuda")
        self.h.attention(layer, q, cu, out, new, work, slots=None if slots is None else i32(slots), lse=lse, scale=scale)
        torch.cuda.synchronize()
        intact()
        intact_l()
        return out, lse


def check_cached(ops, new, kv, page, hq, hk, hd, dt, seed=0, slots=None, layers=1, layer=0, scale=0.0, poison=True):
    n = len(new)
    c = Cache(ops, kv, page, hk, hd, dt, layers=layers, seed=seed)
    if poison:
        # what no slot holds: free pages, and last pages behind their slot's length
        free = (c.refs == 0).nonzero()[:, 0]
        c.k[:, free], c.v[:, free] = math.nan, math.inf
        for s, m in enumerate(kv):
            if m % page:
                p = int(c.tables[s, m // page])
                c.k[:, p, m % page:], c.v[:, p, m % page:] = math.nan, -math.inf
    cu = offsets(new)
    q = rnd(cu[-1] + 2, hq, hd, dt=dt, seed=seed + 5)
    out, lse = c.attend(q, cu, slots=slots, layer=layer, scale=scale)
    for i in range(n):
        a, b = cu[i], cu[i + 1]
        k, v = c.rows(slots[i] if slots else i, layer)
        m = k.shape[0]
        pos = torch.arange(b - a, device="cuda")[:, None] + m - (b - a)
        o, z, tol, tol_z = attention_reference(q[a:b], k, v, torch.arange(m, device="cuda") <= pos,
                                               scale or 1 / math.sqrt(hd))
        close(out[a:b], o, tol)
        close(lse[a:b], z, tol_z)
    assert bool((out[cu[-1]:] == 7).all()) and bool((lse[cu[-1]:] == 7).all())


@pytest.mark.parametrize("dt", [BF16, F16])
@pytest.mark.parametrize("hq,hk,hd", SHAPES)
@pytest.mark.parametrize("page", [16, 64])
def test_cached_tokens(ops, dt, hq, hk, hd, page):
    check_cached(ops, [1] * 9, [1, 2, 15, 16, 17, 128, 129, 300, 777], page, hq, hk, hd, dt, seed=hd)


@pytest.mark.parametrize("page", [16, 32, 64, 128])
@pytest.mark.parametrize("new,kv", [([1], [1]), ([1], [500]), ([1], [20000]), ([3, 0, 1], [3, 40, 1000]),
                                    ([0, 0], [0, 7]), ([64, 65, 130], [64, 700, 1000]), ([300], [5000]),
                                    ([1, 1, 1], [0, 5, 0]), ([5, 200, 9], [2, 130, 9]), ([16] * 20, [400] * 20)])
def test_cached_lengths(ops, page, new, kv):
    """From one token to whole prompts, lengths of zero, and queries that see
    nothing (more of them than the slot has tokens): 0 and -infinity."""
    check_cached(ops, new, kv, page, 8, 2, 128, BF16, seed=page + sum(kv))


def test_cached_layers_slots_and_scale(ops):
    check_cached(ops, [2, 1, 4], [300, 40, 555], 32, 4, 2, 64, F16, layers=3, layer=2, slots=[2, 0, 1], scale=0.3)
    check_cached(ops, [1, 5], [300, 40], 16, 6, 2, 128, BF16, slots=[0, 0])  # one slot named twice


@pytest.mark.parametrize("n", [1, 40, 1500, 3000])
def test_cached_many_sequences(ops, n):
    r = random.Random(n)
    kv = [r.choice([1, 9, 130, 400]) for _ in range(n)]
    check_cached(ops, [1] * n, kv, 16, 2, 1, 64, BF16, seed=n, poison=False)


def test_cached_hint_below_the_truth(ops):
    """max_new steers the split only: a hint that is too small changes nothing."""
    c = Cache(ops, [700, 90], 16, 2, 64, BF16, seed=4)
    q = rnd(300, 4, 64, dt=BF16, seed=8)
    a, la = c.attend(q, [0, 250, 300])
    b, lb = c.attend(q, [0, 250, 300], max_new=1)
    tol = 4 * half_step(BF16) * (a.double().abs() + 1)
    assert bool(((a.double() - b.double()).abs() <= tol).all()) and bool(((la - lb).abs() <= 1e-4).all())


def test_cached_bad_state_stays_in_range(ops):
    """Pages that do not exist read as zeros; lengths, slots and offsets out
    of range write nothing outside the rows of the call."""
    c = Cache(ops, [100, 60], 16, 2, 64, BF16, seed=4, width=8)
    q = rnd(2, 4, 64, dt=BF16, seed=8)
    k, v = c.rows(0)
    for bad in (-1, c.pages, 2 ** 31 - 1, -2 ** 31):
        c.tables[0, 2] = bad
        kk, vv = k.clone(), v.clone()
        kk[32:48], vv[32:48] = 0, 0
        out, _ = c.attend(q, [0, 1, 2])
        o, _, tol, _ = attention_reference(q[:1], kk, vv, torch.ones(1, 100, dtype=torch.bool, device="cuda"), 1 / 8)
        close(out[:1], o, tol)
    for lens in ([2 ** 31 - 1, 60], [-5, 60], [129, 60]):
        c.lens.copy_(i32(lens))
        c.attend(q, [0, 1, 2])
    c.lens.copy_(i32([100, 60]))
    for slots in ([-1, 1], [2, 1], [2 ** 31 - 1, -2 ** 31]):
        c.attend(q, [0, 1, 2], slots=slots)
    for cu in ([0, 1, 300], [-40, 1, 2], [0, 2, 1], [2 ** 31 - 1] * 3):
        c.attend(q, cu, max_new=1)


def test_cached_past_32_bits(ops):
    """Pages whose elements lie past 2^31 and 2^32 from the pool's start."""
    layers, pages, page, hk, hd = 2, 18000, 128, 8, 128  # 2.36e9 elements a layer
    k = torch.empty(layers, pages, page, hk, hd, device="cuda", dtype=BF16)
    v = torch.empty_like(k)
    mine = [17999, 16500, 9, 17000]
    for x, s in ((k, 1), (v, 2)):
        x[1, mine] = rnd(4, page, hk, hd, dt=BF16, seed=s)
    tables, lens = i32([mine]), i32([450])
    refs = torch.zeros(pages, dtype=torch.int32, device="cuda")
    refs[mine] = 1
    h = ops.KvCache(k, v, tables, lens, refs)
    q, out = rnd(3, 16, hd, dt=BF16, seed=3), torch.empty(3, 16, hd, device="cuda", dtype=BF16)
    cu = i32([0, 3])
    nk, nv = rnd(3, hk, hd, dt=BF16, seed=7), rnd(3, hk, hd, dt=BF16, seed=8)
    h.write(1, nk, nv, cu)
    assert torch.equal(k[1, 17000, 450 - 384 - 3:450 - 384], nk) and torch.equal(v[1, 17000, 63:66], nv)
    work = torch.zeros(h.attention_workspace(q, cu, 3), dtype=torch.uint8, device="cuda")
    h.attention(1, q, cu, out, 3, work)
    kk, vv = (x[1, mine].reshape(-1, hk, hd)[:450] for x in (k, v))
    see = torch.arange(450, device="cuda") <= torch.arange(447, 450, device="cuda")[:, None]
    o, _, tol, _ = attention_reference(q, kk, vv, see, 1 / math.sqrt(hd))
    close(out, o, tol)
    # a page moved from there to the front, in the second layer
    status = i32([9, 9])
    h.compact(status)
    assert status.tolist() == [0, 3] and tables.tolist() == [[3, 1, 9, 2]] or sorted(tables[0].tolist()) == [0, 1, 2, 3]
    h.attention(1, q, cu, out, 3, work)
    close(out, o, tol)


# --------------------------------------------------------------------- pages --
class Model:
    """The page operations, one request after the other, on lists."""

    def __init__(self, c):
        self.tables, self.lens, self.refs, self.page = c.tables.tolist(), c.lens.tolist(), c.refs.tolist(), c.page
        self.copies = []

    def take(self):
        p = self.refs.index(0)
        self.refs[p] = 1
        return p

    def free_pages(self):
        return self.refs.count(0)

    def reserve(self, slots, add):
        need = sum(-(-(self.lens[s] + a) // self.page) - -(-self.lens[s] // self.page) for s, a in zip(slots, add))
        if need > self.free_pages():
            return [1, need]
        for s, a in zip(slots, add):
            for j in range(-(-self.lens[s] // self.page), -(-(self.lens[s] + a) // self.page)):
                self.tables[s][j] = self.take()
            self.lens[s] += a
        return [0, need]

    def fork(self, src, dst):
        need = sum(self.lens[s] % self.page > 0 for s in src)
        if need > self.free_pages():
            return [1, need]
        for a, b in zip(src, dst):
            full, rest = divmod(self.lens[a], self.page)
            for j in range(full):
                self.tables[b][j] = self.tables[a][j]
                self.refs[self.tables[a][j]] += 1
            if rest:
                self.tables[b][full] = self.take()
                self.copies.append((self.tables[a][full], self.tables[b][full], rest))
            self.lens[b] = self.lens[a]
        return [0, need]

    def free(self, slots):
        gone = 0
        for s in slots:
            for j in range(-(-self.lens[s] // self.page)):
                p = self.tables[s][j]
                self.refs[p] -= 1
                gone += self.refs[p] == 0
            self.tables[s] = [-1] * len(self.tables[s])
            self.lens[s] = 0
        return [0, gone]

    def compact(self):
        live = [p for p, r in enumerate(self.refs) if r]
        holes = [p for p in range(len(live)) if not self.refs[p]]
        new = dict(zip([p for p in live if p >= len(live)], holes))
        for a, b in new.items():
            self.refs[b], self.refs[a] = self.refs[a], 0
            self.copies.append((a, b, self.page))
        self.tables = [[new.get(p, p) for p in row] for row in self.tables]
        return [0, len(new)]


def same_state(c, m):
    assert c.tables.tolist() == m.tables
    assert c.lens.tolist() == m.lens
    assert c.refs.tolist() == m.refs


@pytest.mark.parametrize("page,layers,seed", [(16, 1, 0), (32, 3, 1), (64, 2, 2), (128, 1, 3)])
def test_pages_against_a_model(ops, page, layers, seed):
    """A long run of random requests, state and contents after each."""
    r = random.Random(seed)
    c = Cache(ops, [], page, 2, 16, BF16, layers=layers, spare=60, seed=seed, width=9, slots=24)
    m = Model(c)
    seen = set()
    for step in range(60):
        k, v = c.k.clone(), c.v.clone()
        m.copies = []
        empty = [s for s in range(24) if m.lens[s] == 0]
        used = [s for s in range(24) if m.lens[s]]
        op = r.choice(["reserve", "reserve", "fork", "fork", "free", "compact"])
        if op == "reserve":
            slots = r.sample(range(24), r.randint(0, 8))
            add = [r.randint(0, min(3 * page, 9 * page - m.lens[s])) for s in slots]
            want = m.reserve(slots, add)
            c.h.reserve(i32(slots), i32(add), c.status)
        elif op == "fork":
            dst = r.sample(empty, r.randint(0, min(6, len(empty))))
            src = [r.choice(used) for _ in dst] if used else []
            dst = dst[:len(src)]
            want = m.fork(src, dst)
            c.h.fork(i32(src), i32(dst), c.status)
        elif op == "free":
            slots = r.sample(range(24), r.randint(0, 6))
            want = m.free(slots)
            c.h.free(i32(slots), c.status)
        else:
            want = m.compact()
            c.h.compact(c.status)
        seen.add((op, want[0]))
        assert c.status.tolist() == want, (step, op)
        same_state(c, m)
        for a, b, n in m.copies:
            k[:, b, :n], v[:, b, :n] = k[:, a, :n], v[:, a, :n]
        assert torch.equal(c.k, k) and torch.equal(c.v, v), (step, op)
        c.k.copy_(rnd(*c.k.shape, dt=BF16, seed=step))
    assert ("fork", 0) in seen and ("reserve", 1) in seen and ("compact", 0) in seen


def test_pages_refused_requests_change_nothing(ops):
    c = Cache(ops, [20, 5, 64, 0], 16, 1, 16, F16, spare=2, seed=1, width=6)
    before = c.state()

    def refused(code=2):
        assert c.status.tolist()[0] == code
        for a, b in zip(c.state(), before):
            assert torch.equal(a, b)
        c.status.fill_(9)
    h, s = c.h, c.status
    h.reserve(i32([0, 0]), i32([1, 1]), s), refused()
    h.reserve(i32([0, 4]), i32([1, 1]), s), refused()
    h.reserve(i32([-1]), i32([1]), s), refused()
    h.reserve(i32([0]), i32([-1]), s), refused()
    h.reserve(i32([1, 2]), i32([3, 33]), s), refused()       # past the row of the table
    h.reserve(i32([0]), i32([2 ** 31 - 1]), s), refused()
    h.reserve(i32([0, 1, 3]), i32([16, 16, 17]), s), refused(1)  # four pages, two are free
    h.fork(i32([0, 1]), i32([3, 3]), s), refused()
    h.fork(i32([0]), i32([1]), s), refused()                 # in use
    h.fork(i32([3]), i32([3]), s), refused()                 # from a slot that it fills
    h.fork(i32([4]), i32([3]), s), refused()
    h.fork(i32([0]), i32([-2 ** 31]), s), refused()
    h.free(i32([0, 1, 0]), s), refused()
    h.free(i32([2 ** 31 - 1]), s), refused()
    h.reserve(i32([]), i32([]), s)
    assert s.tolist() == [0, 0]
    h.free(i32([]), s), h.fork(i32([]), i32([]), s)
    assert s.tolist() == [0, 0]


def test_pages_many(ops):
    """More pages, slots and table entries than one pass of a CTA takes."""
    slots, page = 3000, 16
    c = Cache(ops, [], page, 1, 8, F16, spare=20000, width=40, slots=slots)
    m = Model(c)
    r = random.Random(0)
    order = r.sample(range(slots), 2500)
    add = [r.randint(0, 100) for _ in order]
    want = m.reserve(order, add)
    c.h.reserve(i32(order), i32(add), c.status)
    assert c.status.tolist() == want
    same_state(c, m)
    gone = r.sample(range(slots), 1700)
    want = m.free(gone)
    c.h.free(i32(gone), c.status)
    assert c.status.tolist() == want
    same_state(c, m)
    want = m.compact()
    c.h.compact(c.status)
    assert c.status.tolist() == want and want[1] > 1024
    same_state(c, m)


def test_pages_write(ops):
    """Rows land behind the slot's earlier ones, whatever the strides; a token
    without a place is left out and rows of others stay."""
    c = Cache(ops, [40, 3, 70], 16, 2, 24, BF16, layers=2, seed=3)
    k0, v0 = c.k.clone(), c.v.clone()
    new, slots = [5, 0, 33], [2, 1, 0]
    cu = offsets(new)
    src = rnd(cu[-1] + 4, 6, 24, dt=BF16, seed=4)
    k, v = src[:, 1:3], src[:, 3:5]
    c.h.write(1, k, v, i32(cu), slots=i32(slots))
    for i, s in enumerate(slots):
        kk, vv = c.rows(s, 1)
        n = new[i]
        assert torch.equal(kk[len(kk) - n:], k[cu[i]:cu[i + 1]]) and torch.equal(vv[len(vv) - n:], v[cu[i]:cu[i + 1]])
        for p in range(int(c.lens[s]) - n):  # the earlier ones
            page = int(c.tables[s, p // 16])
            assert torch.equal(c.k[1, page, p % 16], k0[1, page, p % 16])
    assert torch.equal(c.k[0], k0[0]) and torch.equal(c.v[0], v0[0])
    c.k.copy_(k0), c.v.copy_(v0)
    c.tables[2, 4] = c.pages  # where the five would go
    c.h.write(1, k, v, i32([0, 5, 5]), slots=i32([2, 1]))
    c.h.write(1, k, v, i32([0, 5]), slots=i32([7]))
    c.h.write(1, k, v, i32([0, 9]), slots=i32([1]))  # six more than the slot holds: only the last three
    p = int(c.tables[1, 0])
    k0[1, p, :3], v0[1, p, :3] = k[6:9], v[6:9]
    assert torch.equal(c.k, k0) and torch.equal(c.v, v0)


# ----------------------------------------------------------------- together --
def run_texts(ops, c, prefix, texts, hq, hk, hd, dt, cos, sin, seed):
    """Texts behind one prefix, as a host uses the operators: turn, write,
    fork, reserve, attend; returns the outputs of the texts' tokens."""
    s = c.status
    cu_p = offsets([prefix])
    x = rnd(prefix, hq + 2 * hk, hd, dt=dt, seed=seed)
    c.h.reserve(i32([0]), i32([prefix]), s)
    ops.rope(x[:, :hq + hk], torch.arange(prefix, device="cuda", dtype=torch.int32), cos, sin)
    c.h.write(0, x[:, hq:hq + hk], x[:, hq + hk:], i32(cu_p), slots=i32([0]))
    n = len(texts)
    dst = i32(list(range(1, n + 1)))
    c.h.fork(i32([0] * n), dst, s)
    c.h.reserve(dst, i32(texts), s)
    cu = offsets(texts)
    y = rnd(cu[-1], hq + 2 * hk, hd, dt=dt, seed=seed + 1)
    pos = torch.cat([torch.arange(prefix, prefix + t, dtype=torch.int32) for t in texts]).cuda()
    raw = y.clone()
    ops.rope(y[:, :hq + hk], pos, cos, sin)
    c.h.write(0, y[:, hq:hq + hk], y[:, hq + hk:], i32(cu), slots=dst)
    out = torch.empty(cu[-1], hq, hd, device="cuda", dtype=dt)
    cud = i32(cu)
    work = torch.zeros(c.h.attention_workspace(y[:, :hq], cud, max(texts)), dtype=torch.uint8, device="cuda")
    c.h.attention(0, y[:, :hq], cud, out, max(texts), work, slots=dst)
    return x, y, raw, cu, out


@pytest.mark.parametrize("dt,hq,hk,hd", [(BF16, 8, 2, 128), (F16, 6, 3, 64)])
def test_texts_behind_a_shared_prefix(ops, dt, hq, hk, hd):
    """The whole run equals the prompt attention of prefix + text, token by
    token, and one more token per text (single-token form) equals it too."""
    prefix, texts = 45, [7, 1, 130, 64]
    cos, sin = (torch.empty(400, hd // 2, device="cuda") for _ in range(2))
    ops.rope_table(cos, sin, 1e4)
    c = Cache(ops, [], 16, hk, hd, dt, spare=60, width=20, slots=6, seed=1)
    x, y, _, cu, out = run_texts(ops, c, prefix, texts, hq, hk, hd, dt, cos, sin, 3)
    u = half_step(dt)
    for i, t in enumerate(texts):
        row = torch.cat([x, y[cu[i]:cu[i + 1]]])
        q, k, v = row[:, :hq], row[:, hq:hq + hk], row[:, hq + hk:]
        full = torch.empty(prefix + t, hq, hd, device="cuda", dtype=dt)
        ops.attn_prompt(q, k, v, i32([0, prefix + t]), full)
        see = torch.ones(prefix + t, prefix + t, dtype=torch.bool, device="cuda").tril()
        o, _, tol, _ = attention_reference(q, k, v, see, 1 / math.sqrt(hd))
        close(full, o, tol)
        close(out[cu[i]:cu[i + 1]], o[prefix:], tol[prefix:])
        kk, vv = c.rows(i + 1)
        assert torch.equal(kk, k) and torch.equal(vv, v)
    # the prefix is held once: its whole pages by all five slots
    first = c.tables[:5, :prefix // 16]
    assert bool((first == first[0]).all()) and bool((c.refs[first[0].long()] == 5).all())
    # one more token each
    dst = i32([1, 2, 3, 4])
    c.h.reserve(dst, i32([1] * 4), c.status)
    z = rnd(4, hq + 2 * hk, hd, dt=dt, seed=9)
    ops.rope(z[:, :hq + hk], i32([prefix + t for t in texts]), cos, sin)
    cu1 = i32([0, 1, 2, 3, 4])
    c.h.write(0, z[:, hq:hq + hk], z[:, hq + hk:], cu1, slots=dst)
    one = torch.empty(4, hq, hd, device="cuda", dtype=dt)
    work = torch.zeros(c.h.attention_workspace(z[:, :hq], cu1, 1), dtype=torch.uint8, device="cuda")
    c.h.attention(0, z[:, :hq], cu1, one, 1, work, slots=dst)
    for i in range(4):
        k, v = c.rows(i + 1)
        see = torch.ones(1, k.shape[0], dtype=torch.bool, device="cuda")
        o, _, tol, _ = attention_reference(z[i:i + 1, :hq], k, v, see, 1 / math.sqrt(hd))
        close(one[i:i + 1], o, tol)
    assert u > 0


def test_captured_and_replayed(ops):
    """The run of operators as a CUDA graph: replays on new contents equal
    calls, two graphs that share nothing but the cache's shapes included."""
    hq, hk, hd, dt = 8, 2, 64, BF16
    cos, sin = (torch.empty(2000, hd // 2, device="cuda") for _ in range(2))
    ops.rope_table(cos, sin, 1e4)
    c = Cache(ops, [900, 40, 0, 333], 16, hk, hd, dt, spare=80, width=80, seed=2)
    cu, one = i32([0, 1, 2, 3, 4]), i32([1, 1, 1, 1])
    slots = i32([0, 1, 2, 3])
    x, pos = rnd(4, hq + 2 * hk, hd, dt=dt, seed=1), i32([900, 40, 0, 333])
    turned, out = torch.empty_like(x), torch.empty(4, hq, hd, device="cuda", dtype=dt)
    work = torch.zeros(c.h.attention_workspace(x[:, :hq], cu, 1), dtype=torch.uint8, device="cuda")

    def step():
        turned.copy_(x)
        c.h.reserve(slots, one, c.status)
        ops.rope(turned[:, :hq + hk], pos, cos, sin)
        c.h.write(0, turned[:, hq:hq + hk], turned[:, hq + hk:], cu, slots=slots)
        c.h.attention(0, turned[:, :hq], cu, out, 1, work, slots=slots)
        pos.add_(1)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()  # loads the kernels
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        step()
    for i in range(20):  # past a page's end
        x.copy_(rnd(*x.shape, dt=dt, seed=20 + i))
        g.replay()
        assert c.status.tolist()[0] == 0
        assert c.lens.tolist() == [902 + i, 42 + i, 2 + i, 335 + i]
        for s in range(4):
            k, v = c.rows(s)
            assert torch.equal(k[-1], turned[s, hq:hq + hk])
            see = torch.ones(1, k.shape[0], dtype=torch.bool, device="cuda")
            o, _, tol, _ = attention_reference(turned[s:s + 1, :hq], k, v, see, 1 / 8)
            close(out[s:s + 1], o, tol)


def test_streams_and_repeatability(ops):
    """Two streams at once, each with its own workspace, and the same bits
    from every run."""
    c = Cache(ops, [5000, 70, 1200, 9], 16, 2, 128, BF16, seed=6)
    q = rnd(4, 8, 128, dt=BF16, seed=7)
    want, lse = c.attend(q, [0, 1, 2, 3, 4])
    cu = i32([0, 1, 2, 3, 4])
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs, works = [], []
    torch.cuda.synchronize()
    for st in streams:
        with torch.cuda.stream(st):
            work = torch.zeros(c.h.attention_workspace(q, cu, 1), dtype=torch.uint8, device="cuda")
            works.append(work)
            for _ in range(10):
                out = torch.empty_like(q)
                c.h.attention(0, q, cu, out, 1, work)
                outs.append(out)
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)
    # prompts too
    x = rnd(700, 8, 128, dt=BF16, seed=1)
    k, v = x[:, :2], x[:, 2:4]
    a, b = torch.empty_like(x), torch.empty_like(x)
    ops.attn_prompt(x, k, v, i32([0, 300, 700]), a)
    ops.attn_prompt(x, k, v, i32([0, 300, 700]), b, stream=streams[0].cuda_stream)
    torch.cuda.synchronize()
    assert torch.equal(a, b)


def test_host_memory_is_refused(ops):
    from embedcuda import _lib
    x = torch.zeros(4, 2, 64, dtype=BF16)
    cos = torch.zeros(8, 32)
    with pytest.raises(_lib.EcError, match="device memory"):
        ops.rope(x, torch.zeros(4, dtype=torch.int32), cos, cos, stream=0)
    with pytest.raises(_lib.EcError, match="device memory"):
        ops.attn_prompt(x, x, x, torch.tensor([0, 4], dtype=torch.int32), x, stream=0)
