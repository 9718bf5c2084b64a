"""Operators on device tensors: rotary positions, causal attention of packed
prompts, and a paged key / value cache with the attention that reads it
(include/embedcuda.h, "operators on device buffers").

Tensors are anything with torch's interface (``data_ptr()``, ``shape``,
``stride()``, ``dtype``, ``device``); the buffers stay the caller's and nothing
is copied.  Work is enqueued on ``stream`` (a cudaStream_t as int; None: torch's
current stream of the tensors' device) and not waited for.
"""
from __future__ import annotations

import ctypes as C
import sys

from . import _lib

_F32, _BF16, _F16, _I32 = _lib.EC_F32, _lib.EC_BF16, _lib.EC_F16, -1
_NAMES = {"torch.float32": _F32, "torch.bfloat16": _BF16, "torch.float16": _F16, "torch.int32": _I32}
_codes = {}  # the same by dtype object (its name is slow to form on every call)
_fns = {}    # bound C entry points
ROPE_NONE, ROPE_LINEAR, ROPE_LLAMA3, ROPE_YARN = 0, 1, 2, 3
KV_OK, KV_FULL, KV_BAD = 0, 1, 2


def _call(name, *args):
    fn = _fns.get(name)
    if fn is None:
        fn = _fns[name] = getattr(_lib.lib(), name)
    rc = fn(*args)
    if rc < 0:
        _lib.check(rc, name[3:])
    return rc


def _stream(stream, t):
    if stream is not None:
        return stream
    torch = sys.modules.get("torch")
    if torch is None:
        return None
    raw = getattr(torch._C, "_cuda_getCurrentRawStream", None)  # the handle alone, without a Stream object
    return raw(t.get_device()) if raw and t.is_cuda else torch.cuda.current_stream(t.device).cuda_stream


def _kind(t):
    code = _codes.get(t.dtype)
    if code is None:
        code = _codes[t.dtype] = _NAMES.get(str(t.dtype), -2)
    return code


def _code(t, what):
    code = _kind(t)
    if code < 0:
        raise ValueError(f"{what}: dtype {t.dtype} (float32, bfloat16 or float16)")
    return code


def _rows(t, what, heads=None, head_dim=None):
    """(pointer, token stride, head stride) of a [tokens, heads, head_dim] tensor."""
    shape, stride = t.shape, t.stride()
    if len(stride) != 3 or (stride[2] != 1 and shape[2] > 1):
        raise ValueError(f"{what} must be [tokens, heads, head_dim] with adjacent elements")
    if (heads is not None and shape[1] != heads) or (head_dim is not None and shape[2] != head_dim):
        raise ValueError(f"{what} has {shape[1]} heads of {shape[2]}, expected {heads} of {head_dim}")
    return t.data_ptr(), stride[0], stride[1]


def _ints(t, what, size=None, least=0):
    shape = t.shape
    if _kind(t) != _I32 or len(shape) != 1 or not t.is_contiguous():
        raise ValueError(f"{what} must be a contiguous int32 vector")
    if (size is not None and shape[0] != size) or shape[0] < least:
        raise ValueError(f"{what} has {shape[0]} elements, expected {size if size is not None else least}")
    return t.data_ptr()


def _lse(t, tokens, heads):
    if t is None:
        return None
    if _kind(t) != _F32 or t.shape != (tokens, heads) or not t.is_contiguous():
        raise ValueError(f"lse must be a contiguous float32[{tokens}, {heads}]")
    return t.data_ptr()


def _tables(cos, sin):
    shape = cos.shape
    for t in (cos, sin):
        if _kind(t) != _F32 or len(shape) != 2 or not t.is_contiguous():
            raise ValueError("cos and sin must be contiguous float32[positions, rot_dim / 2]")
    if shape != sin.shape:
        raise ValueError(f"cos {tuple(cos.shape)} and sin {tuple(sin.shape)} differ")
    return shape


# keys of rope_scaling that a table is made by (a type has no use for the others'
# keys), and those that say nothing about it (how much of a head is turned is
# the tables' width)
_SCALING = {"rope_type", "type", "factor", "low_freq_factor", "high_freq_factor", "beta_fast", "beta_slow",
            "attention_factor", "original_max_position_embeddings", "finetuned", "partial_rotary_factor"}


def rope_table(cos, sin, theta, scaling=None, stream=None):
    """Fill cos and sin float32[positions, rot_dim / 2].  ``scaling`` is
    config.json's rope_scaling (None, or rope_type linear / llama3 / yarn with
    their keys); a key that would change the table in another way is an error."""
    positions, half = _tables(cos, sin)
    s = {k: v for k, v in (scaling or {}).items() if v is not None}
    kind = s.get("rope_type", s.get("type", "default" if not s else None))
    if s.pop("rope_theta", theta) != theta:
        raise ValueError(f"rope_scaling has another rope_theta than {theta}")
    if s.get("truncate") is True:  # yarn's range in whole pairs
        del s["truncate"]
    unknown = [k for k in s if k not in _SCALING]
    if unknown and kind in ("linear", "llama3", "yarn"):
        raise ValueError(f"rope_scaling {kind} with {', '.join(unknown)}")
    factor, p0, p1, original, amp = 1.0, 0.0, 0.0, 0.0, 0.0
    if kind == "default":
        code = ROPE_NONE
    elif kind == "linear":
        code, factor = ROPE_LINEAR, s["factor"]
    elif kind == "llama3":
        code, factor = ROPE_LLAMA3, s["factor"]
        p0, p1, original = s["low_freq_factor"], s["high_freq_factor"], s["original_max_position_embeddings"]
    elif kind == "yarn":
        code, factor = ROPE_YARN, s["factor"]
        p0, p1, original = s.get("beta_fast", 32.0), s.get("beta_slow", 1.0), s["original_max_position_embeddings"]
        amp = s.get("attention_factor") or 0.0
    else:
        raise ValueError(f"rope_scaling type {kind!r} (linear, llama3 or yarn)")
    _call("ec_rope_table", cos.data_ptr(), sin.data_ptr(), positions, 2 * half, theta, code, factor, p0, p1, original,
          amp, _stream(stream, cos))


def rope(x, pos, cos, sin, out=None, interleaved=False, inverse=False, stream=None):
    """Turn the first 2 * cos.shape[1] elements of every head of x [tokens,
    heads, head_dim] by its token's position (int32[tokens]); into ``out``, or
    in place.  ``inverse`` turns back (the gradient).  Returns the result."""
    positions, half = _tables(cos, sin)
    code = _code(x, "x")
    shape = x.shape
    xr = yr = _rows(x, "x")
    if out is None:
        out = x
    else:
        if _code(out, "out") != code or out.shape != shape:
            raise ValueError(f"out {tuple(out.shape)} {out.dtype} does not match x {tuple(shape)} {x.dtype}")
        yr = _rows(out, "out")
    tokens, heads, hd = shape
    _call("ec_rope", *xr, *yr, code, tokens, heads, hd, 2 * half, 1 if interleaved else 0, 1 if inverse else 0,
          _ints(pos, "pos", tokens), cos.data_ptr(), sin.data_ptr(), positions, _stream(stream, x))
    return out


def attn_prompt(q, k, v, cu, out, lse=None, scale=0.0, stream=None):
    """Causal attention of packed prompts: q, out [tokens, q_heads, head_dim],
    k, v [tokens, kv_heads, head_dim], sequence s the tokens cu[s]:cu[s + 1]
    (int32 on the device); lse float32[tokens, q_heads] or None.  Returns out."""
    tokens, hq, hd = q.shape
    hk = k.shape[1]
    code = _code(q, "q")
    for t, what in ((k, "k"), (v, "v"), (out, "out")):
        if _kind(t) != code:
            raise ValueError(f"{what} is {t.dtype}, q is {q.dtype}")
        if t.shape[0] != tokens:
            raise ValueError(f"{what} has {t.shape[0]} tokens, q has {tokens}")
    _call("ec_attn_prompt", *_rows(q, "q"), *_rows(k, "k", hk, hd), *_rows(v, "v", hk, hd), *_rows(out, "out", hq, hd),
          _lse(lse, tokens, hq), code, tokens, hq, hk, hd, _ints(cu, "cu", least=1), cu.shape[0] - 1, scale,
          _stream(stream, q))
    return out


class KvCache:
    """A paged cache in the caller's tensors: k, v [layers, pages, page_size,
    heads, head_dim] (bfloat16 or float16), tables int32[slots, width], lens
    int32[slots], refs int32[pages].  The object keeps the tensors alive; an
    empty cache has lens and refs 0.  Calls on one cache must be ordered by
    their streams.  Results of the page operations arrive in ``status``
    (int32[2] on the device: KV_OK / KV_FULL / KV_BAD and a page count)."""

    def __init__(self, k, v, tables, lens, refs, work=None):
        if k.dim() != 5 or k.shape != v.shape or k.dtype != v.dtype or not k.is_contiguous() or not v.is_contiguous():
            raise ValueError("k and v must be contiguous [layers, pages, page_size, heads, head_dim] of one type")
        layers, pages, page, heads, hd = k.shape
        if _kind(tables) != _I32 or tables.dim() != 2 or not tables.is_contiguous():
            raise ValueError("tables must be a contiguous int32[slots, width]")
        slots, width = tables.shape
        code = _code(k, "k")
        lens_p, refs_p = _ints(lens, "lens", slots), _ints(refs, "refs", pages)
        size = _lib.check(_lib.lib().ec_kv_work_size(pages, slots), "kv_work_size")
        if work is None:
            work = refs.new_zeros((size + 3) // 4)
        if not work.is_contiguous():
            raise ValueError("work must be contiguous")
        for t, what in ((v, "v"), (tables, "tables"), (lens, "lens"), (refs, "refs"), (work, "work")):
            if t.device != k.device:
                raise ValueError(f"{what} is on {t.device}, k is on {k.device}")
        h = C.c_int()
        _lib.check(_lib.lib().ec_kv_open(k.data_ptr(), v.data_ptr(), code, layers, pages, page, heads, hd,
                                         tables.data_ptr(), slots, width, lens_p, refs_p, work.data_ptr(),
                                         work.numel() * work.element_size(), C.byref(h)), "kv_open")
        self._handle = h.value
        self._keep = (k, v, tables, lens, refs, work)
        self.dtype, self.heads, self.head_dim, self.slots = k.dtype, heads, hd, slots

    def close(self):
        if self._handle:
            _lib.lib().ec_kv_close(self._handle)
        self._handle = 0
        self._keep = ()

    def __del__(self):
        if getattr(self, "_handle", 0) and _lib is not None and _lib._lib is not None:
            self.close()

    def reserve(self, slots, add, status, stream=None):
        """Room for add[i] more tokens in slots[i]."""
        n = slots.shape[0]
        _call("ec_kv_reserve", self._handle, _ints(slots, "slots"), _ints(add, "add", n), n, _ints(status, "status", 2),
              _stream(stream, status))

    def fork(self, src, dst, status, stream=None):
        """Empty slots dst[i] become copies of src[i] (whole pages shared)."""
        n = src.shape[0]
        _call("ec_kv_fork", self._handle, _ints(src, "src"), _ints(dst, "dst", n), n, _ints(status, "status", 2),
              _stream(stream, status))

    def free(self, slots, status, stream=None):
        """Empty the slots."""
        _call("ec_kv_free", self._handle, _ints(slots, "slots"), slots.shape[0], _ints(status, "status", 2),
              _stream(stream, status))

    def compact(self, status, stream=None):
        """Move the pages in use to the front."""
        _call("ec_kv_compact", self._handle, _ints(status, "status", 2), _stream(stream, status))

    def _slots(self, slots, n):
        if slots is not None:
            return _ints(slots, "slots", n)
        if n > self.slots:
            raise ValueError(f"{n} sequences, the cache has {self.slots} slots")
        return None

    def write(self, layer, k, v, cu, slots=None, stream=None):
        """Rows k, v [tokens, heads, head_dim] into `layer`: sequence s is the
        last cu[s + 1] - cu[s] tokens of slots[s] (None: slot s)."""
        tokens, n = k.shape[0], cu.shape[0] - 1
        if k.dtype != self.dtype or v.dtype != self.dtype or v.shape[0] != tokens:
            raise ValueError(f"k and v must be {self.dtype} rows of the same tokens")
        _call("ec_kv_write", self._handle, layer, *_rows(k, "k", self.heads, self.head_dim),
              *_rows(v, "v", self.heads, self.head_dim), tokens, _ints(cu, "cu", least=1), self._slots(slots, n), n,
              _stream(stream, k))

    def attention_workspace(self, q, cu, max_new):
        """Bytes of `attention`'s workspace for these shapes (zero it before its first use)."""
        return _call("ec_attn_cached_work_size", self._handle, q.shape[0], q.shape[1], cu.shape[0] - 1, max_new)

    def attention(self, layer, q, cu, out, max_new, workspace, slots=None, lse=None, scale=0.0, stream=None):
        """Attention of the new tokens q [tokens, q_heads, head_dim] over their
        slots' pages (their own keys and values included).  Returns out."""
        tokens, hq, hd = q.shape
        n = cu.shape[0] - 1
        if q.dtype != self.dtype or out.dtype != self.dtype or out.shape[0] != tokens:
            raise ValueError(f"q and out must be {self.dtype} rows of the same tokens")
        if not workspace.is_contiguous():
            raise ValueError("workspace must be contiguous")
        _call("ec_attn_cached", self._handle, layer, *_rows(q, "q", None, self.head_dim),
              *_rows(out, "out", hq, self.head_dim), _lse(lse, tokens, hq), tokens, hq, _ints(cu, "cu", least=1),
              self._slots(slots, n), n, max_new, scale, workspace.data_ptr(), workspace.nbytes, _stream(stream, q))
        return out
