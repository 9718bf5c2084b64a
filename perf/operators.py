"""The cases on which the operators over device buffers are measured: rotary
positions, causal attention over packed prompts, attention over a paged cache,
and the cache's page operations.  Each has a plain form in elementary torch
operations (``own`` false), the framework's calls (``own`` true) and its
definition in 64 bits (``exact``)."""
import math
import os
import random
import sys

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
SIZE = {"bf16": 2, "f16": 2, "f32": 4}


# ------------------------------------------------------------------ cases --
def listed():
    return [
        # one new token of one sequence, queries and keys in one row (16 + 8
        # heads, the Qwen3-0.6B shape): latency
        {"name": "rope-token", "op": "rope", "tokens": 1, "heads": 24, "head_dim": 128, "rot": 128,
         "dtype": "bf16", "interleaved": False, "inverse": False, "positions": 1024, "scaling": "none",
         "packed": True, "rebuild": False},
        # a batch of prompts at far positions, frequencies scaled by yarn
        {"name": "rope-batch", "op": "rope", "tokens": 65536, "heads": 24, "head_dim": 128, "rot": 128,
         "dtype": "bf16", "interleaved": False, "inverse": False, "positions": 131072, "scaling": "yarn",
         "packed": True, "rebuild": False},
        # the context grows: the table is rebuilt (llama3 frequencies) and
        # part of a 96-wide head turned, adjacent pairs, fp32 gradient
        {"name": "rope-rebuild", "op": "rope", "tokens": 9001, "heads": 12, "head_dim": 96, "rot": 64,
         "dtype": "f32", "interleaved": True, "inverse": True, "positions": 262144, "scaling": "llama3",
         "packed": False, "rebuild": True},
        # a query and a few short texts, head dim 64, seven query heads per
        # key head, an empty sequence among them: latency
        {"name": "prompt-few", "op": "prompt", "seqs": 9, "lo": 0, "hi": 37, "spread": 5, "q_heads": 14,
         "kv_heads": 2, "head_dim": 64, "dtype": "f16", "packed": True},
        # the corpus batch of the Qwen3-0.6B benchmark (128 .. 512 tokens)
        {"name": "prompt-corpus", "op": "prompt", "seqs": 256, "lo": 128, "hi": 512, "spread": 3,
         "q_heads": 16, "kv_heads": 8, "head_dim": 128, "dtype": "bf16", "packed": True},
        # one long document
        {"name": "prompt-long", "op": "prompt", "seqs": 1, "lo": 16384, "hi": 16384, "spread": 0,
         "q_heads": 8, "kv_heads": 2, "head_dim": 128, "dtype": "bf16", "packed": False},
        # one token of one short sequence: latency
        {"name": "cached-token", "op": "cached", "seqs": 1, "new_lo": 1, "new_hi": 1, "past_lo": 499,
         "past_hi": 499, "spread": 0, "page": 16, "q_heads": 16, "kv_heads": 8, "head_dim": 128,
         "dtype": "bf16"},
        # one token for each of a batch of sequences of uneven length
        {"name": "cached-batch", "op": "cached", "seqs": 64, "new_lo": 1, "new_hi": 1, "past_lo": 64,
         "past_hi": 8192, "spread": 2, "page": 16, "q_heads": 32, "kv_heads": 8, "head_dim": 128,
         "dtype": "bf16"},
        # one token of each of three long contexts, odd length, large pages
        {"name": "cached-long", "op": "cached", "seqs": 3, "new_lo": 1, "new_hi": 1, "past_lo": 100003,
         "past_hi": 131001, "spread": 1, "page": 64, "q_heads": 16, "kv_heads": 8, "head_dim": 128,
         "dtype": "f16"},
        # texts behind a cached prefix: the new tokens of every text
        {"name": "cached-texts", "op": "cached", "seqs": 96, "new_lo": 16, "new_hi": 300, "past_lo": 650,
         "past_hi": 700, "spread": 4, "page": 32, "q_heads": 16, "kv_heads": 8, "head_dim": 128,
         "dtype": "bf16"},
        # texts forked off a shared prefix, room for their tokens, and these written
        {"name": "pages-fork", "op": "fork", "layers": 8, "pages": 4096, "page": 16, "kv_heads": 8,
         "head_dim": 128, "dtype": "bf16", "forks": 96, "prefix": 333, "lo": 1, "hi": 300, "spread": 6},
        # half of the sequences gone: the cache's live pages moved together
        {"name": "pages-compact", "op": "compact", "layers": 8, "pages": 4096, "page": 16, "kv_heads": 8,
         "head_dim": 128, "dtype": "f16", "slots": 200, "lo": 1, "hi": 300, "spread": 7},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["rope", "prompt", "cached", "cached", "fork", "compact"])
    kv = rng.choice([1, 2, 3, 4, 8])
    group = rng.choice([1, 2, 3, 4, 5, 7, 8])
    hd = rng.choice([32, 64, 64, 96, 128, 128])
    dt = rng.choice(["bf16", "f16"])
    if op == "rope":
        hd = rng.choice([64, 80, 96, 128, 256])
        rot = rng.choice([hd, hd, hd // 2])
        heads = kv * (group + 1)
        tokens = _log(rng, 1, min(60000, int(1e8 / (heads * hd))))
        return {"op": op, "tokens": tokens, "heads": heads, "head_dim": hd, "rot": rot,
                "dtype": rng.choice(["bf16", "f16", "f32"]), "interleaved": rng.random() < 0.5,
                "inverse": rng.random() < 0.3, "positions": _log(rng, 512, 262144),
                "scaling": rng.choice(["none", "linear", "llama3", "yarn"]),
                "packed": rng.random() < 0.5, "rebuild": rng.random() < 0.25}
    if op == "prompt":
        hi = _log(rng, 1, 6000)
        seqs = max(1, min(300, int(rng.uniform(0.2, 1.0) * 24e6 / (hi * hi * kv * group))))
        seqs = min(seqs, _log(rng, 1, 300))
        return {"op": op, "seqs": seqs, "lo": rng.choice([0, hi // 4, hi]), "hi": hi,
                "spread": rng.randrange(1000), "q_heads": kv * group, "kv_heads": kv, "head_dim": hd,
                "dtype": dt, "packed": rng.random() < 0.6}
    if op == "cached":
        past = _log(rng, 1, 60000)
        seqs = max(1, min(_log(rng, 1, 128), int(1.5e6 / (past * kv))))
        new = 1 if rng.random() < 0.6 else max(1, min(_log(rng, 2, 400), int(3e8 / (seqs * kv * group * (past + 400)))))
        return {"op": op, "seqs": seqs, "new_lo": 1, "new_hi": new, "past_lo": past // rng.choice([1, 3, 20]),
                "past_hi": past, "spread": rng.randrange(1000), "page": rng.choice([16, 32, 64, 128]),
                "q_heads": kv * group, "kv_heads": kv, "head_dim": hd, "dtype": dt}
    page = rng.choice([16, 32, 64])
    base = {"op": op, "layers": rng.randint(1, 8), "pages": _log(rng, 600, 4096) * 16 // page, "page": page,
            "kv_heads": rng.choice([1, 2, 4, 8]), "head_dim": rng.choice([64, 128]), "dtype": dt,
            "lo": 1, "spread": rng.randrange(1000)}
    room = base["pages"] * page
    if op == "fork":
        prefix = _log(rng, 1, 700)
        hi = rng.randint(1, 300)
        forks = max(1, min(_log(rng, 1, 128), (room - prefix) // (hi + 2 * page)))
        return {**base, "forks": forks, "prefix": prefix, "hi": hi}
    hi = rng.randint(1, 400)
    return {**base, "slots": max(1, min(_log(rng, 4, 256), room // (hi + page))), "hi": hi}


def _lengths(n, lo, hi, spread):
    """n lengths in [lo, hi], spread over their logarithm; the first is lo
    and the last hi where there are several."""
    r = random.Random(1000 * spread + n)
    out = [min(hi, max(lo, _log(r, max(1, lo), max(1, hi)))) for _ in range(n)]
    if n > 2:
        out[0], out[-1] = lo, hi
    return out


def _offsets(lens):
    cu = [0]
    for v in lens:
        cu.append(cu[-1] + v)
    return cu


# --------------------------------------------------------------- prepare --
def _i32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


SCALINGS = {
    "none": None,
    "linear": {"rope_type": "linear", "factor": 4.0},
    "llama3": {"rope_type": "llama3", "factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0,
               "original_max_position_embeddings": 8192},
    "yarn": {"rope_type": "yarn", "factor": 4.0, "beta_fast": 32.0, "beta_slow": 1.0,
             "original_max_position_embeddings": 32768},
}
THETA = 1e6


def _table(positions, rot, scaling, dtype=torch.float64):
    """cos and sin [positions, rot / 2]: angles in 64 bits, elementary torch
    operations."""
    dev = "cuda"
    f = THETA ** (-torch.arange(0, rot, 2, dtype=torch.float64, device=dev) / rot)
    s = SCALINGS[scaling]
    amp = 1.0
    if scaling == "linear":
        f = f / s["factor"]
    elif scaling == "llama3":
        orig, lo, hi = s["original_max_position_embeddings"], s["low_freq_factor"], s["high_freq_factor"]
        turns = orig * f / (2 * math.pi)  # rotations within the original context
        keep = ((turns - lo) / (hi - lo)).clamp(0, 1)
        f = (1 - keep) * f / s["factor"] + keep * f
    elif scaling == "yarn":
        orig = s["original_max_position_embeddings"]
        dim = lambda b: rot * math.log(orig / (b * 2 * math.pi)) / (2 * math.log(THETA))  # noqa: E731
        low, high = max(math.floor(dim(s["beta_fast"])), 0), min(math.ceil(dim(s["beta_slow"])), rot - 1)
        i = torch.arange(rot // 2, dtype=torch.float64, device=dev)
        ramp = ((i - low) / max(high - low, 1e-3)).clamp(0, 1)
        f = f / s["factor"] * ramp + f * (1 - ramp)
        amp = 0.1 * math.log(s["factor"]) + 1
    a = torch.arange(positions, dtype=torch.float64, device=dev)[:, None] * f
    return (a.cos() * amp).to(dtype), (a.sin() * amp).to(dtype)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def rnd(*shape, dtype=dt):
        return torch.randn(*shape, device="cuda", dtype=torch.float32, generator=g).to(dtype)

    st = {"case": case}
    if case["op"] == "rope":
        t, h, hd = case["tokens"], case["heads"], case["head_dim"]
        # packed: the query and key heads of rows that hold value heads too
        x = rnd(t, h + 4, hd)[:, :h] if case["packed"] else rnd(t, h, hd)
        st["x"], st["y"] = x, torch.zeros(t, h, hd, device="cuda", dtype=dt)
        st["pos"] = torch.randint(0, case["positions"], (t,), device="cuda", dtype=torch.int32, generator=g)
        st["cos"], st["sin"] = _table(case["positions"], case["rot"], case["scaling"], torch.float32)
        return st
    if case["op"] == "prompt":
        lens = _lengths(case["seqs"], case["lo"], case["hi"], case["spread"])
        cu = _offsets(lens)
        t, hq, hk, hd = cu[-1], case["q_heads"], case["kv_heads"], case["head_dim"]
        if case["packed"]:  # query, key and value heads in one row
            x = rnd(t, hq + 2 * hk, hd)
            st["q"], st["k"], st["v"] = x[:, :hq], x[:, hq:hq + hk], x[:, hq + hk:]
        else:
            st["q"], st["k"], st["v"] = rnd(t, hq, hd), rnd(t, hk, hd), rnd(t, hk, hd)
        st["cu"], st["longest"] = _i32(cu), max(lens)
        st["out"] = torch.zeros(t, hq, hd, device="cuda", dtype=dt)
        st["lse"] = torch.zeros(t, hq, device="cuda", dtype=torch.float32)
        return st
    page, hk, hd = case["page"], case["kv_heads"], case["head_dim"]
    if case["op"] == "cached":
        new, kv = _cached_lengths(case)
        cu = _offsets(new)
        need = [-(-n // page) for n in kv]
        width = max(need)
        total = sum(need) + 3
        perm = torch.randperm(total, device="cuda", generator=g).to(torch.int32)  # pages in no order
        tables = torch.full((len(kv), width), -1, dtype=torch.int32, device="cuda")
        col = torch.arange(width, device="cuda")
        first = torch.tensor(_offsets(need)[:-1], device="cuda")
        have = col < torch.tensor(need, device="cuda")[:, None]
        tables = torch.where(have, perm[(first[:, None] + col).clamp(max=total - 1)], tables)
        st.update(q=rnd(cu[-1], case["q_heads"], hd), k=rnd(1, total, page, hk, hd), v=rnd(1, total, page, hk, hd),
                  cu=_i32(cu), lens=_i32(kv), tables=tables, most=max(new),
                  refs=torch.ones(total, dtype=torch.int32, device="cuda"),
                  out=torch.zeros(cu[-1], case["q_heads"], hd, device="cuda", dtype=dt),
                  lse=torch.zeros(cu[-1], case["q_heads"], device="cuda", dtype=torch.float32))
        return st
    # page operations: a cache in use
    n = case["forks"] + 1 if case["op"] == "fork" else case["slots"]
    lens = _lengths(n, case["lo"], case["hi"], case["spread"])
    st["k"], st["v"] = rnd(case["layers"], case["pages"], page, hk, hd), rnd(case["layers"], case["pages"], page, hk, hd)
    st["status"] = torch.zeros(2, dtype=torch.int32, device="cuda")
    if case["op"] == "fork":
        width = -(-(case["prefix"] + case["hi"]) // page)
        p = -(-case["prefix"] // page)
        perm = torch.randperm(case["pages"], device="cuda", generator=g)[:p].to(torch.int32)
        st["tables"] = torch.full((n, width), -1, dtype=torch.int32, device="cuda")
        st["tables"][0, :p] = perm  # slot 0 holds the prefix
        st["lens"] = _i32([case["prefix"]] + [0] * (n - 1))
        st["refs"] = torch.zeros(case["pages"], dtype=torch.int32, device="cuda")
        st["refs"][perm.long()] = 1
        st["src"], st["dst"] = _i32([0] * (n - 1)), _i32(list(range(1, n)))
        add = lens[1:]
        st["add"], st["cu"] = _i32(add), _i32(_offsets(add))
        st["new_k"], st["new_v"] = rnd(sum(add), hk, hd), rnd(sum(add), hk, hd)
        return st
    need = [-(-v // page) for v in lens]
    width = max(need)
    # the sequences came one after the other; every second one is gone
    first = torch.tensor(_offsets(need)[:-1], device="cuda")
    col = torch.arange(width, device="cuda")
    live = torch.arange(n, device="cuda") % 2 == 1
    have = (col < torch.tensor(need, device="cuda")[:, None]) & live[:, None]
    st["tables"] = torch.where(have, first[:, None] + col, -1).to(torch.int32)
    st["lens"] = torch.where(live, torch.tensor(lens, device="cuda"), 0).to(torch.int32)
    st["refs"] = torch.zeros(case["pages"], dtype=torch.int32, device="cuda")
    st["refs"][st["tables"][have].long()] = 1
    st["tables0"], st["refs0"] = st["tables"].clone(), st["refs"].clone()
    return st


def _cached_lengths(case):
    new = _lengths(case["seqs"], case["new_lo"], case["new_hi"], case["spread"])
    past = _lengths(case["seqs"], case["past_lo"], case["past_hi"], case["spread"] + 1)
    return new, [a + b for a, b in zip(new, past)]


# ------------------------------------------------------------------- run --
def run(state):
    op = state["case"]["op"]
    if own:
        return {"rope": _own_rope, "prompt": _own_prompt, "cached": _own_cached, "fork": _own_fork,
                "compact": _own_compact}[op](state)
    return {"rope": _plain_rope, "prompt": _plain_prompt, "cached": _plain_cached, "fork": _plain_fork,
            "compact": _plain_compact}[op](state)


# ---- the framework's calls
def _ops():
    path = os.path.join(os.getcwd(), "lisp-embed_b200")
    if path not in sys.path:
        sys.path.insert(1, path)
    from embedcuda import ops
    return ops


def _own_rope(s):
    ops, c = _ops(), s["case"]
    if c["rebuild"]:
        ops.rope_table(s["cos"], s["sin"], THETA, SCALINGS[c["scaling"]])
    ops.rope(s["x"], s["pos"], s["cos"], s["sin"], out=s["y"], interleaved=c["interleaved"], inverse=c["inverse"])
    return {"y": s["y"], "cos": s["cos"], "sin": s["sin"]} if c["rebuild"] else {"y": s["y"]}


def _own_prompt(s):
    _ops().attn_prompt(s["q"], s["k"], s["v"], s["cu"], s["out"], lse=s["lse"])
    return {"out": s["out"], "lse": s["lse"]}


def _cache(s):
    """The handle that a program keeps beside its cache."""
    if "cache" not in s:
        s["cache"] = _ops().KvCache(s["k"], s["v"], s["tables"], s["lens"], s["refs"])
    return s["cache"]


def _own_cached(s):
    cache = _cache(s)
    if "work" not in s:  # kept between calls, as the cache is
        s["work"] = torch.zeros(cache.attention_workspace(s["q"], s["cu"], s["most"]), dtype=torch.uint8, device="cuda")
    cache.attention(0, s["q"], s["cu"], s["out"], max_new=s["most"], lse=s["lse"], workspace=s["work"])
    return {"out": s["out"], "lse": s["lse"]}


def _pages_out(s):
    return {n: s[n] for n in ("k", "v", "tables", "lens", "refs", "status")}


def _own_fork(s):
    cache = _cache(s)
    cache.free(s["dst"], s["status"])  # what the texts before held
    cache.fork(s["src"], s["dst"], s["status"])
    cache.reserve(s["dst"], s["add"], s["status"])
    cache.write(0, s["new_k"], s["new_v"], s["cu"], slots=s["dst"])
    return _pages_out(s)


def _own_compact(s):
    s["tables"].copy_(s["tables0"])  # the cache as it was, to move the same pages again
    s["refs"].copy_(s["refs0"])
    _cache(s).compact(s["status"])
    return _pages_out(s)


# ---- plain forms
def _plain_rope(s):
    c = s["case"]
    if c["rebuild"]:
        cos, sin = _table(c["positions"], c["rot"], c["scaling"], torch.float32)
        s["cos"].copy_(cos)
        s["sin"].copy_(sin)
    x, rot = s["x"].float(), c["rot"]
    p = s["pos"].long()
    co, si = s["cos"][p][:, None], s["sin"][p][:, None]
    if c["inverse"]:
        si = -si
    if c["interleaved"]:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        turned = torch.stack([a * co - b * si, b * co + a * si], -1).flatten(-2)
    else:
        a, b = x[..., :rot // 2], x[..., rot // 2:rot]
        turned = torch.cat([a * co - b * si, b * co + a * si], -1)
    s["y"].copy_(torch.cat([turned, x[..., rot:]], -1))
    return {"y": s["y"], "cos": s["cos"], "sin": s["sin"]} if c["rebuild"] else {"y": s["y"]}


def _attend(q, k, v, see):
    """q [n, Q, Hq, d], k and v [n, K, Hkv, d], see [n, Q, K]: the attention
    in 32 bits and its log-sum-exp [n, Q, Hq]; a row that sees nothing is 0
    and -inf."""
    n, nq, hq, d = q.shape
    hk = k.shape[2]
    qh = q.view(n, nq, hk, hq // hk, d).permute(0, 2, 3, 1, 4).reshape(n, hk, -1, d)  # rows (group, query)
    sc = torch.matmul(qh, k.permute(0, 2, 3, 1)).view(n, hk, hq // hk, nq, -1)
    sc.mul_(1.0 / math.sqrt(d)).masked_fill_(~see[:, None, None], -math.inf)
    m = sc.amax(-1, keepdim=True)
    m = torch.where(m == -math.inf, torch.zeros_like(m), m)
    p = sc.sub_(m).exp_()
    l = p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(n, hk, -1, p.shape[-1]), v.permute(0, 2, 1, 3)).view(n, hk, hq // hk, nq, d)
    o = o / torch.where(l == 0, torch.ones_like(l), l)
    lse = (m + l.log()).squeeze(-1)
    return o.permute(0, 3, 1, 2, 4).reshape(n, nq, hq, d), lse.permute(0, 3, 1, 2).reshape(n, nq, hq)


def _spread_out(cu, width, total):
    """Rows of a padded [n, width] view of packed rows, and (sequence, row)
    of every packed row."""
    cu = cu.long()
    at = cu[:-1, None] + torch.arange(width, device="cuda")
    t = torch.arange(total, device="cuda")
    seq = torch.searchsorted(cu, t, right=True) - 1
    return at.clamp(max=max(total - 1, 0)), seq, t - cu[seq]


def _plain_prompt(s):
    q, width = s["q"], s["longest"]
    at, seq, row = _spread_out(s["cu"], width, q.shape[0])
    pos = torch.arange(width, device="cuda")
    n = s["cu"].shape[0] - 1
    see = (pos[:, None] >= pos).expand(n, width, width)  # a row past its sequence is not read back
    o, lse = _attend(q[at].float(), s["k"][at].float(), s["v"][at].float(), see)
    s["out"].copy_(o[seq, row])
    s["lse"].copy_(lse[seq, row])
    return {"out": s["out"], "lse": s["lse"]}


def _plain_cached(s):
    q, width = s["q"], s["most"]
    at, seq, row = _spread_out(s["cu"], width, q.shape[0])
    kv = s["lens"].long()
    new = (s["cu"][1:] - s["cu"][:-1]).long()
    pages = s["tables"].long().clamp(min=0)
    k, v = s["k"][0][pages].flatten(1, 2).float(), s["v"][0][pages].flatten(1, 2).float()
    key = torch.arange(k.shape[1], device="cuda")
    v.masked_fill_((key >= kv[:, None])[..., None, None], 0.0)  # what a page holds past its sequence is not read
    pos = (kv - new)[:, None] + torch.arange(width, device="cuda")
    see = (key <= pos[..., None]) & (key < kv[:, None, None])
    o, lse = _attend(q[at].float(), k, v, see)
    s["out"].copy_(o[seq, row])
    s["lse"].copy_(lse[seq, row])
    return {"out": s["out"], "lse": s["lse"]}


def _lowest_free(refs):
    """Pages in the order in which they are given out: free ones first, the
    lowest first."""
    return torch.sort((refs != 0).to(torch.int32), stable=True).indices


def _plain_reserve(s, slots, add):
    page = s["case"]["page"]
    have = s["lens"][slots].long()
    old, want = (have + page - 1) // page, (have + add + page - 1) // page
    need = want - old
    off = torch.cumsum(need, 0) - need
    col = torch.arange(s["tables"].shape[1], device="cuda")
    fresh = (col >= old[:, None]) & (col < want[:, None])
    rank = (off[:, None] + col - old[:, None]).clamp(0, s["refs"].shape[0] - 1)
    got = _lowest_free(s["refs"])[rank]
    s["tables"][slots] = torch.where(fresh, got.to(torch.int32), s["tables"][slots])
    s["refs"].index_add_(0, got.flatten(), fresh.flatten().to(torch.int32))
    s["lens"][slots] = (have + add).to(torch.int32)
    s["status"][0], s["status"][1] = 0, need.sum()


def _plain_free(s, slots):
    page = s["case"]["page"]
    col = torch.arange(s["tables"].shape[1], device="cuda")
    rows = s["tables"][slots]
    used = col < ((s["lens"][slots].long() + page - 1) // page)[:, None]
    s["refs"].index_add_(0, rows.clamp(min=0).flatten().long(), -used.flatten().to(torch.int32))
    s["tables"][slots] = -1
    s["lens"][slots] = 0


def _plain_fork(s):
    page = s["case"]["page"]
    src, dst = s["src"].long(), s["dst"].long()
    _plain_free(s, dst)
    # whole pages are shared, the last one, if it is not full, is copied
    n = s["lens"][src].long()
    full, rest = n // page, n % page
    col = torch.arange(s["tables"].shape[1], device="cuda")
    rows = s["tables"][src].long()
    shared = col < full[:, None]
    part = (col == full[:, None]) & (rest > 0)[:, None]
    need = (rest > 0).long()
    got = _lowest_free(s["refs"])[(torch.cumsum(need, 0) - need).clamp(max=s["refs"].shape[0] - 1)]
    s["refs"].index_add_(0, rows.clamp(min=0).flatten(), shared.flatten().to(torch.int32))
    s["refs"].index_add_(0, got, need.to(torch.int32))
    s["tables"][dst] = torch.where(shared, rows, torch.where(part, got[:, None], -1)).to(torch.int32)
    s["lens"][dst] = n.to(torch.int32)
    frm = rows.gather(1, full.clamp(max=rows.shape[1] - 1)[:, None])[:, 0].clamp(min=0)
    to = torch.where(rest > 0, got, frm)
    row = (torch.arange(page, device="cuda") < rest[:, None])[..., None, None]
    s["k"][:, to] = torch.where(row, s["k"][:, frm], s["k"][:, to])
    s["v"][:, to] = torch.where(row, s["v"][:, frm], s["v"][:, to])
    _plain_reserve(s, dst, s["add"].long())
    # the new tokens' rows into their pages
    t = torch.arange(s["new_k"].shape[0], device="cuda")
    cu = s["cu"].long()
    i = torch.searchsorted(cu, t, right=True) - 1
    at = s["lens"][dst[i]].long() - (cu[i + 1] - t)
    where = s["tables"][dst[i], at // page].long()
    s["k"][0][where, at % page] = s["new_k"]
    s["v"][0][where, at % page] = s["new_v"]
    return _pages_out(s)


def _plain_compact(s):
    s["tables"].copy_(s["tables0"])
    s["refs"].copy_(s["refs0"])
    live = s["refs"] > 0
    total = live.sum()
    ids = torch.arange(live.shape[0], device="cuda")
    hole, high = ~live & (ids < total), live & (ids >= total)
    # the lowest hole takes the lowest page above, and so on
    nth_hole = torch.sort((~hole).to(torch.int32), stable=True).indices
    nth_high = torch.sort((~high).to(torch.int32), stable=True).indices
    moved = ids < high.sum()
    frm, to = torch.where(moved, nth_high, ids[-1]), torch.where(moved, nth_hole, ids[-1])
    new = ids.clone()
    new.index_add_(0, torch.where(moved, nth_high, ids), torch.where(moved, nth_hole - nth_high, 0))
    s["k"][:, to] = s["k"][:, frm]
    s["v"][:, to] = s["v"][:, frm]
    s["tables"].copy_(torch.where(s["tables"] >= 0, new[s["tables"].long().clamp(min=0)].to(torch.int32), s["tables"]))
    refs = torch.where(ids < total, s["refs"], 0)
    refs.index_add_(0, to, torch.where(moved, s["refs"][frm], 0))
    s["refs"].copy_(torch.where(ids < total, refs, 0))
    s["status"][0], s["status"][1] = 0, high.sum()
    return _pages_out(s)


# ------------------------------------------------------------------ work --
def work(case):
    sz = SIZE[case["dtype"]]
    if case["op"] == "rope":
        n = case["tokens"] * case["heads"] * case["head_dim"]
        rows = min(case["tokens"], case["positions"])
        table = case["positions"] * case["rot"] * 4 if case["rebuild"] else rows * case["rot"] * 4
        return {"bytes": 2 * n * sz + case["tokens"] * 4 + table,
                "flops": 3 * case["tokens"] * case["heads"] * case["rot"]}
    if case["op"] == "prompt":
        lens = _lengths(case["seqs"], case["lo"], case["hi"], case["spread"])
        t, hd = sum(lens), case["head_dim"]
        return {"bytes": t * (2 * case["q_heads"] + 2 * case["kv_heads"]) * hd * sz + t * case["q_heads"] * 4,
                "flops": 4 * case["q_heads"] * hd * sum(v * (v + 1) // 2 for v in lens)}
    hk, hd = case["kv_heads"], case["head_dim"]
    if case["op"] == "cached":
        new, kv = _cached_lengths(case)
        t = sum(new)
        pairs = sum(a * (b - a) + a * (a + 1) // 2 for a, b in zip(new, kv))
        return {"bytes": 2 * sum(kv) * hk * hd * sz + t * case["q_heads"] * (2 * hd * sz + 4),
                "flops": 4 * case["q_heads"] * hd * pairs}
    row = 2 * hk * hd * sz  # a token's keys and values in one layer
    page = case["page"]
    if case["op"] == "fork":
        add = _lengths(case["forks"] + 1, case["lo"], case["hi"], case["spread"])[1:]
        part = case["prefix"] % page
        tables = 4 * case["forks"] * -(-(case["prefix"] + case["hi"]) // page)
        return {"bytes": (part + case["forks"] * part) * row * case["layers"] + 2 * sum(add) * row + 3 * tables
                + 4 * case["pages"], "flops": sum(add)}
    lens = _lengths(case["slots"], case["lo"], case["hi"], case["spread"])
    first, live = 0, []
    for i, v in enumerate(lens):
        need = -(-v // page)
        if i % 2:
            live += range(first, first + need)
        first += need
    moves = sum(p >= len(live) for p in live)
    tables = case["slots"] * max(-(-v // page) for v in lens) * 4
    return {"bytes": 2 * moves * page * row * case["layers"] + 2 * tables + 8 * case["pages"], "flops": 1 + moves}


# ----------------------------------------------------------------- exact --
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "rope":
        return _exact_rope(case, s)
    if case["op"] in ("prompt", "cached"):
        return _exact_attention(case, s)
    return _exact_pages(case, s)


def _exact_rope(case, s):
    """Pairs as complex numbers: y = x e^(+-i angle)."""
    rot, x = case["rot"], s["x"].double()
    out = {}
    if case["rebuild"]:
        f = [THETA ** (-2.0 * i / rot) for i in range(rot // 2)]
        sc, amp = SCALINGS[case["scaling"]], 1.0
        if case["scaling"] == "linear":
            f = [v / sc["factor"] for v in f]
        if case["scaling"] == "llama3":
            orig = sc["original_max_position_embeddings"]
            for i, v in enumerate(f):
                wave = 2 * math.pi / v
                if wave > orig / sc["low_freq_factor"]:
                    f[i] = v / sc["factor"]
                elif wave >= orig / sc["high_freq_factor"]:
                    part = (orig / wave - sc["low_freq_factor"]) / (sc["high_freq_factor"] - sc["low_freq_factor"])
                    f[i] = (1 - part) * v / sc["factor"] + part * v
        if case["scaling"] == "yarn":
            orig = sc["original_max_position_embeddings"]
            at = [rot * math.log(orig / (b * 2 * math.pi)) / (2 * math.log(THETA)) for b in (32.0, 1.0)]
            low, high = max(math.floor(at[0]), 0), min(math.ceil(at[1]), rot - 1)
            for i, v in enumerate(f):
                ramp = min(1.0, max(0.0, (i - low) / max(high - low, 1e-3)))
                f[i] = v / sc["factor"] * ramp + v * (1 - ramp)
            amp = 0.1 * math.log(sc["factor"]) + 1
        w = torch.tensor(f, dtype=torch.float64, device="cuda")
        ang = torch.outer(torch.arange(case["positions"], dtype=torch.float64, device="cuda"), w)
        turn = torch.polar(torch.full_like(ang, amp), ang)
        out["cos"], out["sin"] = turn.real.clone(), turn.imag.clone()
        turn = turn[s["pos"].long()]
    else:
        turn = torch.complex(s["cos"][s["pos"].long()].double(), s["sin"][s["pos"].long()].double())
    if case["inverse"]:
        turn = turn.conj()
    half = rot // 2
    i0 = torch.arange(half, device="cuda") * (2 if case["interleaved"] else 1)
    i1 = i0 + (1 if case["interleaved"] else half)
    z = torch.complex(x[..., i0], x[..., i1]) * turn[:, None]
    y = x.clone()
    y[..., i0], y[..., i1] = z.real, z.imag
    return {"y": y, **out}


def _exact_attention(case, s):
    """Sequence by sequence and key head by key head, in 64 bits."""
    hq, hk, hd = case["q_heads"], case["kv_heads"], case["head_dim"]
    group = hq // hk
    cu = s["cu"].tolist()
    out = torch.zeros(cu[-1], hq, hd, dtype=torch.float64, device="cuda")
    lse = torch.full((cu[-1], hq), -math.inf, dtype=torch.float64, device="cuda")
    for i, (a, b) in enumerate(zip(cu, cu[1:])):
        if a == b:
            continue
        if case["op"] == "prompt":
            k, v = s["k"][a:b].double(), s["v"][a:b].double()
        else:
            n = int(s["lens"][i])
            pages = s["tables"][i, :-(-n // case["page"])].long()
            k = s["k"][0, pages].reshape(-1, hk, hd)[:n].double()
            v = s["v"][0, pages].reshape(-1, hk, hd)[:n].double()
        n, m = k.shape[0], b - a
        hidden = torch.triu(torch.ones(m, n, dtype=torch.bool, device="cuda"), n - m + 1)
        for h in range(hq):
            sc = (s["q"][a:b, h].double() @ k[:, h // group].T) / math.sqrt(hd)
            sc.masked_fill_(hidden, -math.inf)
            z = torch.logsumexp(sc, 1)
            lse[a:b, h] = z
            out[a:b, h] = torch.exp(sc - z[:, None]) @ v[:, h // group]
    return {"out": out, "lse": lse}


def _exact_pages(case, s):
    """One request after the other, on lists."""
    page = case["page"]
    tables, lens, refs = s["tables"].tolist(), s["lens"].tolist(), s["refs"].tolist()
    k, v = s["k"].double(), s["v"].double()
    if case["op"] == "compact":
        live = [p for p, r in enumerate(refs) if r]
        holes = [p for p in range(len(live)) if not refs[p]]
        high = [p for p in live if p >= len(live)]
        new = dict(zip(high, holes))
        for a, b in new.items():
            k[:, b], v[:, b] = k[:, a], v[:, a]
            refs[b], refs[a] = refs[a], 0
        tables = [[new.get(p, p) for p in row] for row in tables]
        status = [0, len(high)]
    else:
        def take():
            p = refs.index(0)
            refs[p] = 1
            return p

        for a, b in zip(s["src"].tolist(), s["dst"].tolist()):
            full, rest = divmod(lens[a], page)
            for j in range(full):
                tables[b][j] = tables[a][j]
                refs[tables[a][j]] += 1
            if rest:
                tables[b][full] = take()
                k[:, tables[b][full], :rest] = k[:, tables[a][full], :rest]
                v[:, tables[b][full], :rest] = v[:, tables[a][full], :rest]
            lens[b] = lens[a]
        given = 0
        for b, n in zip(s["dst"].tolist(), s["add"].tolist()):
            for j in range(-(-lens[b] // page), -(-(lens[b] + n) // page)):
                tables[b][j] = take()
                given += 1
            lens[b] += n
        cu = s["cu"].tolist()
        where = [tables[b][p // page] * page + p % page
                 for i, b in enumerate(s["dst"].tolist())
                 for p in range(lens[b] - (cu[i + 1] - cu[i]), lens[b])]
        at = torch.tensor(where, device="cuda")
        k[0].flatten(0, 1)[at] = s["new_k"].double()
        v[0].flatten(0, 1)[at] = s["new_v"].double()
        status = [0, given]
    return {"k": k, "v": v, "tables": _i32(tables), "lens": _i32(lens), "refs": _i32(refs), "status": _i32(status)}
