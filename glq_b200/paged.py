"""Between a decoder's q/k/v and output projections: rotary positions, a paged cache of keys and values, attention over it.

``rotary_table`` holds the frequencies of a model's rotary positions; ``rotary`` rotates heads by them, ``paged_append`` puts new keys
(rotated on the way) and values into a paged cache and rotates their queries in the same launch, ``paged_attention`` lets queries, one of a
sequence or a chunk of many, attend to what the cache holds.  A cache is a pair of tensors (pages, page_size, kv_heads, head_dim) of
bf16 or fp16, in any order of strides with a head's values one behind the other; a page's number is its place in the first dimension.  The
operators run on the current stream of their tensors' device, take a workspace from torch's allocator where they need one, read
nothing back and can be captured into a CUDA graph.  They have no gradients.  No counterpart in the reference, which leaves attention to the
framework that serves the model.
"""
from __future__ import annotations

import ctypes as C
import math
from typing import Optional

import torch

from . import _lib
from .mx4 import _DTYPES, _call, _cuda, _dtype, _same_device

_RAN_ON: set = set()                # devices whose status word a call may have set
_INTEGERS = (torch.int32, torch.int64)
_CACHE_TYPES = {t: _DTYPES[t] for t in (torch.bfloat16, torch.float16)}
_NONE = (0, 0)                      # strides of what is not there


class Rotary:
    """Frequencies of rotary positions (``rotary_table``): ``turns`` int64 (pairs,) on the device, the fraction of a turn that a pair makes per
    position in units of 2^-64; ``scale`` on cosine and sine; ``interleaved``: neighbouring values make a pair, else values half of the
    rotated part apart; ``dim``: values of a head that are rotated.  The attributes cannot be set."""
    __slots__ = ("turns", "scale", "interleaved", "dim", "_desc", "_ref", "_index")

    def __init__(self, turns, scale=1.0, interleaved=False):
        _cuda(turns, "turns")
        if turns.dtype != torch.int64 or turns.dim() != 1 or not turns.numel() or not turns.is_contiguous():
            raise ValueError(f"glq_b200: turns must be int64 (pairs,), got {tuple(turns.shape)} of {turns.dtype}")
        desc = _lib.RotaryDesc(turns.data_ptr(), turns.numel(), bool(interleaved), float(scale))
        for name, value in zip(self.__slots__, (turns, float(scale), bool(interleaved), 2 * turns.numel(), desc, C.byref(desc), turns.get_device())):
            object.__setattr__(self, name, value)

    def __setattr__(self, name, value):
        raise AttributeError(f"glq_b200: {name} of a rotary table cannot be set")


def _frequencies(dim, base, scaling):
    """(radians per position of every pair, scale on cosine and sine), in 64 bits on the host."""
    f = float(base) ** (-torch.arange(0, dim, 2, dtype=torch.float64) / dim)
    if scaling is None:
        return f, 1.0
    kind = scaling.get("rope_type", scaling.get("type"))

    def need(key):
        if key not in scaling:
            raise ValueError(f"glq_b200: {kind!r} rotary scaling needs {key!r}")
        return scaling[key]

    if kind == "default":
        return f, 1.0
    if kind not in ("linear", "llama3", "yarn"):
        raise ValueError(f'glq_b200: rotary scaling is "linear", "llama3" or "yarn", not {kind!r}')
    factor = float(need("factor"))
    if kind == "linear":
        return f / factor, 1.0
    old = float(need("original_max_position_embeddings"))
    if kind == "llama3":
        # pairs that turn at least `high` times within the old context stay, those of at most `low` turns are stretched
        low, high = float(need("low_freq_factor")), float(need("high_freq_factor"))
        keep = ((old * f / (2 * math.pi) - low) / (high - low)).clamp(0, 1)
        return f / factor * (1 - keep) + f * keep, 1.0

    def magnitude(mscale):
        return 0.1 * mscale * math.log(factor) + 1.0 if factor > 1 else 1.0

    def pair(turns):          # the pair that makes so many turns within the old context
        return dim * math.log(old / (turns * 2 * math.pi)) / (2 * math.log(base))

    lo, hi = pair(float(scaling.get("beta_fast") or 32.0)), pair(float(scaling.get("beta_slow") or 1.0))
    if scaling.get("truncate", True):
        lo, hi = math.floor(lo), math.ceil(hi)
    lo, hi = max(lo, 0), min(hi, dim - 1)
    stretched = ((torch.arange(dim // 2, dtype=torch.float64) - lo) / max(hi - lo, 0.001)).clamp(0, 1)
    scale = scaling.get("attention_factor")
    if scale is None:
        if scaling.get("mscale") and scaling.get("mscale_all_dim"):
            scale = magnitude(scaling["mscale"]) / magnitude(scaling["mscale_all_dim"])
        else:
            scale = magnitude(1.0)
    return f / factor * stretched + f * (1 - stretched), float(scale)


def rotary_table(dim=None, *, base=None, scaling=None, interleaved=False, inv_freq=None, scale=None, device=None) -> Rotary:
    """Frequencies base^(-2 i / dim) of ``dim`` rotated values (even), made once for a model.  ``scaling``: a dict as model
    configurations hold it, "rope_type" "linear", "llama3" or "yarn" with its factors.  ``base``: its "rope_theta" by default, else 10000.  ``inv_freq``: radians per position of every pair, in
    place of dim, base and scaling.  ``scale``: factor on cosine and sine in place of the scaling's own.  Frequencies are held in 64
    bits: an angle is off by position * (2^-52 of the frequency given + 2^-65 of a turn) at most, and by 2^-26 of a turn where it becomes fp32."""
    own = 1.0
    if inv_freq is not None:
        if dim is not None and dim != 2 * inv_freq.numel() or scaling is not None:
            raise ValueError("glq_b200: inv_freq comes in place of dim, base and scaling")
        f = inv_freq.detach().to("cpu", torch.float64).reshape(-1)
    else:
        if dim is None or dim < 2 or dim % 2:
            raise ValueError(f"glq_b200: an even number of values is rotated, not {dim}")
        if base is None:
            base = (scaling or {}).get("rope_theta") or 10000.0
        f, own = _frequencies(dim, base, scaling)
    if not f.numel() or not bool(torch.isfinite(f).all()):
        raise ValueError("glq_b200: frequencies must be finite")
    # fractions of a turn in 2^-64, as signed integers, the nearest ones (whole turns per position make no difference at whole positions; half a
    # turn is the same forth and back)
    turns = f / (2 * math.pi)
    turns = [round(math.ldexp(p, 64)) for p in (turns - turns.round()).tolist()]
    turns = torch.tensor([t - 2 ** 64 if t == 2 ** 63 else t for t in turns], dtype=torch.int64)
    device = torch.device("cuda" if device is None else device)
    if device.type != "cuda":
        raise RuntimeError("glq_b200: a rotary table is used on a CUDA device (there is no CPU path)")
    return Rotary(turns.to(device), own if scale is None else scale, interleaved)


def _device_of(x, name, index=None):
    """The device a tensor is on, which is ``index`` if that is given.  (One call instead of three: -1 is the host's, others have none.)"""
    try:
        own = x.get_device()
    except AttributeError:
        own = -1
    if own < 0:
        _cuda(x, name)
    if index is not None and own != index:
        raise ValueError(f"glq_b200: {name} is on {x.device}, expected cuda:{index}")
    return own


def _heads(x, name, index=None):
    """x (tokens, heads, head_dim) with a head's values one behind the other, its shape, strides and span: the addresses from its first value to
    behind its last.  On the device ``index`` if that is given."""
    _device_of(x, name, index)
    shape = x.shape
    if len(shape) != 3:
        raise ValueError(f"glq_b200: {name} is (tokens, heads, head_dim), got {tuple(shape)}")
    stride = x.stride()
    if stride[2] != 1 and shape[2] > 1:
        x = x.contiguous()
        stride = x.stride()
    return x, shape, stride, _span(x, shape, stride)


def _span(x, shape, stride):
    first = x.data_ptr()
    t, h, d = shape
    if not (t and h and d):
        return first, first
    return first, first + ((t - 1) * stride[0] + (h - 1) * stride[1] + d) * x.itemsize


def _result(out, x, shape, stride, span, name):
    """Where a tensor's result goes, its strides and span: a new tensor, or the given ``out``, which has x's shape, type and device, no two
    values in one place, and is x itself or lies apart from it."""
    if out is None:
        t, h, d = shape
        own = (h * d, d, 1)
        return torch.empty_like(x) if stride == own else torch.empty_strided(shape, own, dtype=x.dtype, device=x.device), own, None
    _same_device(out, x, name)
    if out.shape != shape or out.dtype != x.dtype:
        raise ValueError(f"glq_b200: {name} must be {tuple(shape)} of {x.dtype}, got {tuple(out.shape)} of {out.dtype}")
    t, h, d = shape
    own = out.stride()
    (a, m), (b, n) = sorted(((own[0], t), (own[1], h)))
    if d > 1 and own[2] != 1 or m > 1 and a < d or n > 1 and b < d or m > 1 and n > 1 and b < a * (m - 1) + d:
        raise ValueError(f"glq_b200: {name} needs a head's values one behind the other and rows that do not overlap, got strides {own}")
    at = _span(out, shape, own)
    if _meet(span, at) and not (span[0] == at[0] and own == stride) and _rows_meet(span, shape, stride, at, shape, own, x):
        raise ValueError(f"glq_b200: {name} overlaps its input without being it")
    return out, own, at


def _meet(a, b):
    """Do two spans have an address in common?"""
    return a[0] < b[1] and b[0] < a[1]


def _rows_meet(a, shape, stride, b, other, own, x):
    """The same of rows: those of one wider matrix (parts of a merged projection) lie within each other's span and may be apart all the same."""
    if not _meet(a, b):
        return False
    step, size = stride[0], x.itemsize
    long, wide = ((s[1] - 1) * t[1] + s[2] for s, t in ((shape, stride), (other, own)))
    if step != own[0] or shape[0] < 2 or long > step or wide > step:
        return True
    apart = (b[0] - a[0]) % (step * size)
    return apart < long * size or apart + wide * size > step * size


def _integers(t, index, name, count):
    """Are they int64 (else int32)?"""
    _device_of(t, name, index)
    dtype = t.dtype
    if dtype not in _INTEGERS or t.shape != (count,) or not t.is_contiguous():
        raise ValueError(f"glq_b200: {name} must be {count} int32 or int64 values, got {tuple(t.shape)} of {dtype}")
    return dtype is torch.int64


def _check_table(table, index, head_dim):
    if table.__class__ is not Rotary:
        raise ValueError("glq_b200: table is what rotary_table returns")
    if table._index != index:
        raise ValueError(f"glq_b200: the rotary table is on {table.turns.device}, expected cuda:{index}")
    if table.dim > head_dim:
        raise ValueError(f"glq_b200: {table.dim} rotated values in heads of {head_dim}")


def rotary(x, positions, table: Rotary, *, out=None) -> torch.Tensor:
    """x (tokens, heads, head_dim) of bf16, fp16 or fp32 with the first ``table.dim`` values of every head rotated by its token's
    position (int32 or int64, (tokens,); negative ones rotate back), computed in fp32 and rounded once; the other values as they are.
    ``out``: where the result goes, x itself too."""
    x, shape, stride, span = _heads(x, "x")
    dt = _dtype(x.dtype, "x")
    tokens, heads, dim = shape
    _check_table(table, x.get_device(), dim)
    wide = _integers(positions, table._index, "positions", tokens)
    out, own, _ = _result(out, x, shape, stride, span, "out")
    if tokens and heads:
        _call(table._index, "rotary", _lib.load().glqb_rotary, table._ref, span[0], dt, stride[0], stride[1], out.data_ptr(), own[0], own[1], tokens, heads, dim,
              positions.data_ptr(), wide)
    return out


def _cache(keys, values):
    """The C description of a cache, checked, its device, shape, type, and the spans of its two tensors."""
    index = _device_of(keys, "key_cache")
    _device_of(values, "value_cache", index)
    shape, dtype = keys.shape, keys.dtype
    if len(shape) != 4 or values.shape != shape or values.dtype != dtype:
        raise ValueError(f"glq_b200: key_cache and value_cache are (pages, page_size, kv_heads, head_dim) of one type, got {tuple(keys.shape)} of {keys.dtype} and "
                         f"{tuple(values.shape)} of {values.dtype}")
    kind = _CACHE_TYPES.get(dtype)
    if kind is None:
        raise ValueError(f"glq_b200: a cache is bf16 or fp16, not {dtype}")
    pages, size, heads, dim = shape
    if pages < 1 or heads < 1 or dim < 8 or dim > 128 or dim % 8 or size < 8 or size & (size - 1):
        raise ValueError(f"glq_b200: a cache of {tuple(shape)}: pages of a power of two rows, 8 at least, heads of a multiple of 8 values, 128 at most")
    (kp, kr, kh, kd), (vp, vr, vh, vd) = keys.stride(), values.stride()
    if pages == 1:
        kp = vp = 0
    if heads == 1:
        kh = vh = 0
    first, other = keys.data_ptr(), values.data_ptr()
    if kd != 1 or vd != 1 or (first | other) & 15 or (kp | kr | kh | vp | vr | vh) & 7:
        raise ValueError(f"glq_b200: key_cache and value_cache must lie on 16 bytes, strides of 8 values, a head's values one behind the other; got strides {keys.stride()} and "
                         f"{values.stride()}")
    desc = _lib.pack_cache(first, other, kp, kr, kh, vp, vr, vh, pages, size, heads, dim, kind)
    pages, size, heads = pages - 1, size - 1, heads - 1
    return (desc, index, shape, dtype, (first, first + 2 * (pages * kp + size * kr + heads * kh + dim)), (other, other + 2 * (pages * vp + size * vr + heads * vh + dim)))


def paged_append(key, value, key_cache, value_cache, slots, *, positions=None, table: Optional[Rotary] = None, query=None, out=None):
    """Puts the keys and values (tokens, kv_heads, head_dim) of new tokens into the cache, in place: token t's into row ``slots[t]`` =
    page * page_size + row (int32 or int64); a slot outside the cache, -1 for one, leaves the cache alone, as for tokens that pad a batch.
    The slots within the cache are all different, and keys and values do not share addresses (they may lie between one another's, as in one tensor).  With ``table`` and ``positions`` (tokens,) the keys are rotated on the way, and so is ``query``
    (tokens, heads, head_dim) if it is given: to a new tensor or to ``out`` (the query itself too), which is returned.  Keys, values and
    queries are of the cache's type, or fp32."""
    desc, index, cache, dtype, kspan, vspan = _cache(key_cache, value_cache)
    key, shape, ks, at_key = _heads(key, "key", index)
    value, value_shape, vs, at_value = _heads(value, "value", index)
    tokens, kv_heads, dim = shape
    if value_shape != shape or kv_heads != cache[2] or dim != cache[3]:
        raise ValueError(f"glq_b200: keys of {tuple(shape)} and values of {tuple(value_shape)} for a cache of {tuple(cache)}")
    kind = key.dtype
    if value.dtype != kind or (kind != dtype and kind != torch.float32):
        raise ValueError(f"glq_b200: keys and values are of the cache's type, {dtype}, or fp32, got {kind} and {value.dtype}")
    slots_wide, positions_wide, at_positions, turn = _integers(slots, index, "slots", tokens), False, 0, None
    if (table is None) != (positions is None):
        raise ValueError("glq_b200: table and positions come together")
    if table is not None:
        _check_table(table, index, dim)
        positions_wide, at_positions, turn = _integers(positions, index, "positions", tokens), positions.data_ptr(), table._ref
    heads, at_query, at_out, qs, os = 0, None, None, _NONE, _NONE
    if query is None:
        if out is not None:
            raise ValueError("glq_b200: out belongs to query")
    else:
        if table is None:
            raise ValueError("glq_b200: query is here to be rotated: table and positions are needed")
        given = out is not None
        query, query_shape, qs, at_query = _heads(query, "query", index)
        heads = query_shape[1]
        if query_shape[0] != tokens or query_shape[2] != dim or query.dtype != kind:
            raise ValueError(f"glq_b200: queries of {tuple(query_shape)}, {query.dtype}, beside keys of {tuple(shape)}, {kind}")
        out, os, at_out = _result(out, query, query_shape, qs, at_query, "out")
        if given and (_rows_meet(at_key, shape, ks, at_out, query_shape, os, key) or _rows_meet(at_value, shape, vs, at_out, query_shape, os, key)):
            raise ValueError("glq_b200: out overlaps key or value")
    for name, at in (("key", at_key), ("value", at_value), ("query", at_query), ("out", at_out)):
        if at is not None and (at[0] < kspan[1] and kspan[0] < at[1] or at[0] < vspan[1] and vspan[0] < at[1]):
            raise ValueError(f"glq_b200: {name} overlaps the cache")
    if tokens:
        a = _lib.pack_append(at_key[0], at_value[0], at_query[0] if at_query is not None else 0, out.data_ptr() if out is not None else 0, ks[0], ks[1], vs[0], vs[1], qs[0],
                                 qs[1], os[0], os[1], tokens, slots.data_ptr(), at_positions, slots_wide, positions_wide, _DTYPES[kind], heads)
        _call(index, "paged_append", _lib.load().glqb_paged_append, desc, a, turn)
    return out


def paged_attention(query, key_cache, value_cache, pages, lengths, *, query_offsets=None, max_query_len=None, scale=None, causal=True, window=0, out=None):
    """Attention of the newest tokens of every sequence over a paged cache that holds their keys and values already.

    ``query`` (tokens, heads, head_dim) of the cache's type, the heads a multiple of the cache's: query head h reads key head
    h // (heads // kv_heads).  ``lengths`` (sequences,): keys of every sequence, those of the new tokens among them, in the pages that
    ``pages`` (sequences, columns) int32 names in order.  ``query_offsets`` (sequences + 1,): rows query_offsets[s] .. query_offsets[s + 1] - 1 are
    the last ones of sequence s, ascending; None: one row per sequence.  A query sees the keys up to its own (``causal``, else to its
    sequence's last), from ``window`` - 1 in front of its own on (0: from the first).  ``scale`` (positive): of the scores, head_dim ** -0.5 by default.
    ``max_query_len``: what no sequence has more rows than, if the program knows it; the faster kernel is chosen by it.
    Integers are int32 or int64 and stay on the device: lengths are held to 0 .. columns * page_size, offsets to 0 .. tokens; a page
    outside the cache reads as zeros.  Rows that see no key are zero.  Rows of no sequence (in front of query_offsets[0], behind the last) are zero in a
    new result and stay as they are in a given ``out``.  Sums and softmax in fp32, weights rounded to the cache's type for the product with the values, as
    is the result; what lies in the cache where no query looks, NaN included, changes nothing.  The same call gives the same bits."""
    desc, index, cache, dtype, kspan, vspan = _cache(key_cache, value_cache)
    query, shape, qs, span = _heads(query, "query", index)
    tokens, heads, dim = shape
    if dim != cache[3] or query.dtype != dtype or heads < 1 or heads % cache[2]:
        raise ValueError(f"glq_b200: queries of {tuple(shape)}, {query.dtype}, over a cache of {tuple(cache)}, {dtype}")
    _device_of(pages, "pages", index)
    table = pages.shape
    if pages.dtype != torch.int32 or len(table) != 2 or (pages.stride(1) != 1 and table[1] > 1):
        raise ValueError(f"glq_b200: pages must be int32 (sequences, columns), a row's entries one behind the other, got {tuple(table)} of {pages.dtype}")
    seqs = table[0]
    lengths_wide, offsets_wide, at_offsets = _integers(lengths, index, "lengths", seqs), False, 0
    if query_offsets is not None:
        offsets_wide, at_offsets = _integers(query_offsets, index, "query_offsets", seqs + 1), query_offsets.data_ptr()
    elif tokens != seqs:
        raise ValueError(f"glq_b200: {tokens} queries of {seqs} sequences need query_offsets")
    if max_query_len is None:
        max_query_len = tokens if query_offsets is not None else 1
    elif max_query_len < 0:
        raise ValueError(f"glq_b200: max_query_len is {max_query_len}")
    if scale is None:
        scale = dim ** -0.5
    elif not (scale > 0.0 and math.isfinite(scale)):
        raise ValueError(f"glq_b200: scale is a positive number, not {scale}")
    window = int(window or 0)
    if not 0 <= window < 2 ** 31:
        raise ValueError(f"glq_b200: a window of {window} keys")
    fresh = out is None
    out, os, at_out = _result(out, query, shape, qs, span, "out")
    if not fresh and (_meet(at_out, span) or _meet(at_out, kspan) or _meet(at_out, vspan)):
        raise ValueError("glq_b200: out overlaps the queries or the cache")
    if tokens:
        if span[0] & 15 or qs[0] & 7 or qs[1] & 7 or not (qs[0] and qs[1]):          # (strides of 0: expanded)
            query = query.clone(memory_format=torch.contiguous_format)
            qs = query.stride()
        a = _lib.pack_attention(query.data_ptr(), out.data_ptr(), qs[0], qs[1], os[0], os[1], tokens, pages.data_ptr(), pages.stride(0), lengths.data_ptr(), at_offsets, lengths_wide,
                                    offsets_wide, seqs, table[1], heads, bool(causal), window, fresh and query_offsets is not None, min(max_query_len, tokens), scale)
        lib = _lib.load()
        size = _workspace(lib, index, desc, a)
        ws = torch.empty_strided((size,), (1,), dtype=torch.uint8, device=query.device)
        _call(index, "paged_attention", lib.glqb_paged_attention, desc, a, ws.data_ptr(), size)
        _RAN_ON.add(index)
    return out


def _workspace(lib, index, cache, call):
    """Bytes of workspace of a call; 0 from the library is a refusal, which the call itself words."""
    cuda = torch._C
    before = cuda._cuda_getDevice()
    if before == index:
        return lib.glqb_paged_attention_workspace_bytes(cache, call)
    cuda._cuda_setDevice(index)
    try:
        return lib.glqb_paged_attention_workspace_bytes(cache, call)
    finally:
        cuda._cuda_setDevice(before)


def paged_check_status() -> None:
    """Synchronise the devices that attention ran on and raise RuntimeError (code GLQB_E_DEVICE) if a bounded wait in it gave up since
    the last call: the results of that run are invalid."""
    for index in sorted(_RAN_ON):
        _call(index, "paged status", lambda stream: _lib.load().glqb_paged_status(None))
