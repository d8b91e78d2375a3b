"""Rotary positions, paged append and attention without a GPU: the oracle against itself, the ABI's structure, the refusals, the list of work."""
import ctypes
import math
import os
import subprocess

import pytest
import torch

import paged_oracle as O

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def lib():
    from glq_b200 import _lib, build
    build.build()
    return _lib.load()


def test_oracle_rotates_by_the_angle():
    x = torch.randn(3, 2, 8, dtype=torch.float64)
    f = torch.tensor([1.0, 0.25], dtype=torch.float64)
    pos = torch.tensor([0, 3, -2])
    for interleaved in (False, True):
        y, _ = O.rotate(x, pos, f, 1.0, interleaved)
        a, b = ((0, 2), (1, 3)) if interleaved is False else ((0, 1), (2, 3))
        for i, (u, v) in enumerate((a, b)):
            z = torch.complex(x[..., u], x[..., v]) * torch.polar(torch.ones(3, dtype=torch.float64), pos * f[i])[:, None]
            assert torch.allclose(y[..., u], z.real, atol=1e-14) and torch.allclose(y[..., v], z.imag, atol=1e-14)
        assert torch.equal(y[0], x[0]) and torch.equal(y[..., 4:], x[..., 4:])


def test_oracle_attention_is_softmax_over_what_is_seen():
    g = torch.Generator().manual_seed(1)
    keys, values = (torch.randn(3, 8, 1, 8, generator=g).half() for _ in range(2))
    q = torch.randn(5, 2, 8, generator=g, dtype=torch.float64)
    pages = torch.tensor([[2, 0]])
    y, _ = O.attend(q, keys, values, pages, [11], [0, 5], window=4)
    k, v = torch.cat((keys[2], keys[0]))[:11, 0].double(), torch.cat((values[2], values[0]))[:11, 0].double()
    back = torch.arange(6, 11)[:, None] - torch.arange(11)[None]
    z = torch.einsum("qhd,kd->hqk", q, k) / math.sqrt(8) + torch.where((back >= 0) & (back < 4), 0.0, -math.inf)
    assert torch.allclose(y, torch.einsum("hqk,kd->qhd", torch.softmax(z, -1), v))


def test_struct_layouts_match_header(tmp_path):
    from glq_b200 import _lib
    pairs = [("GlqbRotary", _lib.RotaryDesc), ("GlqbPagedCache", _lib.PagedCacheDesc), ("GlqbPagedAppend", _lib.PagedAppendDesc), ("GlqbPagedAttention", _lib.PagedAttentionDesc)]
    lines = "".join(f'printf("%zu ", sizeof({c}));' + "".join(f'printf("%zu ", __builtin_offsetof({c}, {f[0]}));' for f in d._fields_) for c, d in pairs)
    src, exe = tmp_path / "s.c", tmp_path / "s"
    src.write_text('#include <stdio.h>\n#include "glq_b200.h"\nint main(){' + lines + "}")
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)], check=True)
    out = [int(v) for v in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()]
    assert out == [v for _, d in pairs for v in [ctypes.sizeof(d)] + [getattr(d, f[0]).offset for f in d._fields_]]


def test_packed_descriptions_are_the_structures():
    from glq_b200 import _lib
    for desc, pack in ((_lib.PagedCacheDesc, _lib.pack_cache), (_lib.PagedAppendDesc, _lib.pack_append), (_lib.PagedAttentionDesc, _lib.pack_attention)):
        values = [0.5 if t is ctypes.c_float else 3 + i for i, (_, t) in enumerate(desc._fields_)]
        assert pack(*values) == bytes(desc(*values))


def test_c_entries_refuse_before_any_cuda_call(lib):
    from glq_b200 import _lib
    p = 4096                                                    # never dereferenced: each call is refused

    def refused(rc, code, text):
        assert rc == code and text in lib.glqb_last_error().decode(), (rc, lib.glqb_last_error())

    def rotary(r=(p, 4, 0, 1.0), x=p, dt=1, out=p, tokens=2, heads=3, dim=64, pos=p):
        return lib.glqb_rotary(ctypes.byref(_lib.RotaryDesc(*r)), x, dt, 192, 64, out, 192, 64, tokens, heads, dim, pos, 1, None)

    refused(rotary(dt=3), -1, "dtype")
    refused(rotary(tokens=-1), -1, "-1 tokens")
    refused(rotary(dim=2000), -1, "2000 values")
    refused(rotary(x=None), -1, "null")
    refused(rotary(out=p + 1), -1, "aligned")
    refused(rotary(r=(None, 4, 0, 1.0)), -1, "turns")
    refused(rotary(r=(p, 33, 0, 1.0)), -1, "33 pairs")
    refused(rotary(r=(p, 0, 0, 1.0)), -1, "0 pairs")
    refused(rotary(pos=p + 4), -1, "aligned")
    assert rotary(tokens=0) == 0 and rotary(heads=0) == 0

    cache = dict(keys=p, values=p, key_page=2048, key_row=128, key_head=64, value_page=2048, value_row=128, value_head=64, pages=10, page_size=16, kv_heads=2, head_dim=64, dtype=1)

    def append(r=(p, 4, 0, 1.0), c={}, **kw):
        a = dict(key=p, value=p, key_token=128, key_head=64, value_token=128, value_head=64, tokens=3, slots=p, positions=p, slots_are_int64=1, positions_are_int64=1, dtype=1)
        a.update(kw)
        return lib.glqb_paged_append(ctypes.byref(_lib.PagedCacheDesc(**{**cache, **c})), ctypes.byref(_lib.PagedAppendDesc(**a)), ctypes.byref(_lib.RotaryDesc(*r)) if r else None, None)

    def attention(ws=p, size=1 << 40, c={}, **kw):
        a = dict(query=p, out=p, query_token=256, query_head=64, out_token=256, out_head=64, tokens=3, page_table=p, page_stride=4, lengths=p, offsets=None, sequences=3,
                 page_columns=4, heads=4, causal=1, scale=0.1, max_query_len=1)
        a.update(kw)
        return lib.glqb_paged_attention(ctypes.byref(_lib.PagedCacheDesc(**{**cache, **c})), ctypes.byref(_lib.PagedAttentionDesc(**a)), ws, size, None)

    for call in (append, attention):
        refused(call(c=dict(dtype=2)), -1, "fp16 or bf16")
        refused(call(c=dict(page_size=24)), -1, "24 rows")
        refused(call(c=dict(page_size=4)), -1, "4 rows")
        refused(call(c=dict(head_dim=136)), -1, "136 values")
        refused(call(c=dict(head_dim=12)), -1, "12 values")
        refused(call(c=dict(kv_heads=0)), -1, "0 heads")
        refused(call(c=dict(pages=1 << 31)), -1, "pages")
        refused(call(c=dict(values=None)), -1, "null")
        refused(call(c=dict(key_row=124)), -1, "multiples of 8")
        refused(call(c=dict(values=p + 8)), -1, "16 bytes")
        for wrong in (dict(key_page=0), dict(value_row=0), dict(key_head=56), dict(value_row=64), dict(key_page=2040), dict(key_page=128, key_row=1024)):
            refused(call(c=wrong), -1, "overlap")
    refused(append(dtype=0), -1, "type")
    refused(append(tokens=-1), -1, "-1 tokens")
    refused(append(slots=None), -1, "null")
    refused(append(query=p, query_out=p, heads=2, r=None), -1, "rotated")
    refused(append(r=(p, 40, 0, 1.0)), -1, "40 pairs")
    refused(append(value=p + 1), -1, "aligned")
    assert append(tokens=0) == 0
    refused(attention(heads=3), -1, "3 query heads")
    refused(attention(tokens=1 << 29), -1, "too many")
    refused(attention(sequences=(1 << 20) + 1), -1, "sequences")
    refused(attention(page_columns=1 << 27), -1, "per sequence")
    for scale in (0.0, -1.0, math.nan, math.inf):
        refused(attention(scale=scale), -1, "positive")
    refused(attention(window=-1), -1, "window")
    refused(attention(out=None), -1, "null")
    refused(attention(lengths=None), -1, "null")
    refused(attention(page_table=None), -1, "null")
    refused(attention(query=p + 8), -1, "16 bytes")
    refused(attention(query_token=260), -1, "multiples of 8")
    refused(attention(ws=p + 4), -1, "aligned")
    assert attention(tokens=0, out=None) == 0


def _append_refusal(lib, keys, values, key_strides, value_strides, pages, size, heads, dim):
    """What a call says of caches at these addresses.  It has too many tokens for a launch, wherever it runs."""
    from glq_b200 import _lib
    cache = _lib.PagedCacheDesc(keys, values, *key_strides, *value_strides, pages, size, heads, dim, 1)
    a = _lib.PagedAppendDesc(key=4096, value=4096, key_token=128, key_head=64, value_token=128, value_head=64, tokens=1 << 40, slots=4096, slots_are_int64=1, dtype=1)
    assert lib.glqb_paged_append(ctypes.byref(cache), ctypes.byref(a), None, None) < 0
    return lib.glqb_last_error().decode()


def test_append_refuses_keys_and_values_in_one_place(lib):
    """Two threads would write each value.  Against every address of both, for keys and values that lie between one another in all manners."""
    import itertools
    import random
    rng = random.Random(3)
    p, found = 1 << 40, {True: 0, False: 0}

    def taken(strides, counts, dim, at):
        return {at + sum(i * s for i, s in zip(ix, strides)) + e for ix in itertools.product(*(range(n) for n in counts)) for e in range(dim)}

    for trial in range(600):
        counts, dim = (rng.randint(1, 3), 8, rng.randint(1, 3)), rng.choice([8, 16])
        order, strides, reach = rng.sample(range(3), 3), [0, 0, 0], dim
        for i in order:
            strides[i] = reach + 8 * rng.choice([0, 0, 1, dim // 8, reach // 8])
            reach = strides[i] * (counts[i] - 1) + reach if counts[i] > 1 else reach
        shift = 8 * rng.randint(-reach // 8 - 2, reach // 8 + 2) if rng.random() < 0.6 else rng.choice(strides) - rng.choice([0, 0, 8]) * rng.choice([-1, 1])
        shift = shift // 8 * 8
        mine = taken(strides, counts, dim, 0)
        meet = any(a + shift in mine for a in mine)
        said = _append_refusal(lib, p, p + 2 * shift, strides, strides, *counts, dim)
        assert ("share" in said) == meet, (counts, dim, strides, shift, said)
        found[meet] += 1
    assert min(found.values()) > 100
    # of different strides: pages that lie beside one another's, or caches that do
    rows, heads = (4096, 128, 64), (4096, 64, 1024)
    for shift, meet in ((2048, False), (-2048, False), (2048 + 4096 * 3, False), (1024, True), (-1024, True), (0, True), (4096 * 10, False), (4096 * 9 + 2048, False), (4096 * 9 - 64, True), (-4096 * 10, False)):
        assert ("share" in _append_refusal(lib, p, p + 2 * shift, rows, heads, 10, 16, 2, 64)) == meet, shift
    far = (1 << 37, 128, 64)                                      # (addresses beyond 64 bits)
    assert "share" in _append_refusal(lib, p, p + 64, far, far, (1 << 31) - 1, 16, 2, 64)
    assert "share" not in _append_refusal(lib, p, p + 4096, far, far, (1 << 31) - 1, 16, 2, 64)


def _table(monkeypatch, dim=32, **kw):
    """A rotary table on the host (its device is not looked at here)."""
    from glq_b200 import paged
    monkeypatch.setattr(paged, "_cuda", lambda t, name: None)
    real = torch.device
    monkeypatch.setattr(paged.torch, "device", lambda d: type("D", (), {"type": "cuda"})() if d == "cuda" else real(d))
    monkeypatch.setattr(torch.Tensor, "to", lambda self, *a, _to=torch.Tensor.to, **k: self if a and not isinstance(a[0], (str, torch.dtype, real)) else _to(self, *a, **k))
    table = paged.rotary_table(dim, **kw)
    monkeypatch.undo()
    return table


def test_table_holds_fractions_of_a_turn(monkeypatch):
    t = _table(monkeypatch, 8, base=100.0)
    for i, v in enumerate(t.turns.tolist()):
        want = 100.0 ** (-2 * i / 8) / (2 * math.pi)
        assert abs((v % 2 ** 64) / 2 ** 64 - want) <= 2.0 ** -52
    assert t.dim == 8 and t.scale == 1.0 and not t.interleaved
    # a frequency beyond a turn per position, and a negative one, wrap
    t = _table(monkeypatch, None, inv_freq=torch.tensor([2 * math.pi * 3.75, -2 * math.pi * 0.25, 2 * math.pi * 0.5]))
    for v, want in zip(t.turns.tolist(), (0.75, 0.75, 0.5)):
        assert abs((v % 2 ** 64) / 2 ** 64 - want) < 1e-6
    with pytest.raises(AttributeError, match="cannot be set"):
        t.scale = 2.0


def test_table_is_rounded(monkeypatch):
    """Of slow pairs, whose frequency's 53 bits end below 2^-64 turns, the nearest number of units is held."""
    from fractions import Fraction
    f = torch.tensor([2.0 ** -40 * 1.7, 2.0 ** -50 * 1.3, -2.0 ** -45 * 1.1, 2.0 ** -66, 1.0], dtype=torch.float64)
    t = _table(monkeypatch, None, inv_freq=f)
    for v, p in zip(t.turns.tolist(), (f / (2 * math.pi)).tolist()):
        off = (v - Fraction(p) * 2 ** 64) % 2 ** 64
        assert min(off, 2 ** 64 - off) <= Fraction(1, 2), (v, p)


def test_base_in_the_scaling(monkeypatch):
    """Configurations may hold a model's base beside its scaling: it is taken where no other is given."""
    plain = _table(monkeypatch, 64, base=500000.0).turns
    assert torch.equal(_table(monkeypatch, 64, scaling={"rope_type": "default", "rope_theta": 500000.0}).turns, plain)
    assert torch.equal(_table(monkeypatch, 64, base=500000, scaling={"rope_type": "default", "rope_theta": 500000.0}).turns, plain)
    yarn = {"rope_type": "yarn", "factor": 4.0, "original_max_position_embeddings": 32768}
    assert torch.equal(_table(monkeypatch, 64, scaling={**yarn, "rope_theta": 5e5}).turns, _table(monkeypatch, 64, base=5e5, scaling=yarn).turns)
    assert torch.equal(_table(monkeypatch, 64, scaling=yarn).turns, _table(monkeypatch, 64, base=10000.0, scaling=yarn).turns)
    assert torch.equal(_table(monkeypatch, 64, base=10000.0, scaling={**yarn, "rope_theta": 5e5}).turns, _table(monkeypatch, 64, scaling=yarn).turns)


@pytest.mark.parametrize("name,kw,dim", [("linear", dict(factor=4.0), 64), ("llama3", dict(factor=8.0, low_freq_factor=1.0, high_freq_factor=4.0, original_max_position_embeddings=8192), 128),
                                         ("yarn", dict(factor=4.0, beta_fast=32.0, beta_slow=1.0, original_max_position_embeddings=32768), 128)])
def test_scalings_of_long_contexts(monkeypatch, name, kw, dim):
    base = 500000.0
    t = _table(monkeypatch, dim, base=base, scaling={"rope_type": name, **kw})
    got = [(v % 2 ** 64) / 2 ** 64 * 2 * math.pi for v in t.turns.tolist()]
    for i, f in enumerate(got):
        plain = base ** (-2 * i / dim)
        if name == "linear":
            want = plain / 4
        else:
            old, length = kw["original_max_position_embeddings"], 2 * math.pi / plain
            if name == "llama3":
                smooth = (old / length - 1.0) / 3.0
                want = plain if length < old / 4 else plain / 8 if length > old else (1 - smooth) * plain / 8 + smooth * plain
            else:
                lo, hi = (dim * math.log(old / (r * 2 * math.pi)) / (2 * math.log(base)) for r in (32.0, 1.0))
                ramp = min(1.0, max(0.0, (i - math.floor(lo)) / (math.ceil(hi) - math.floor(lo))))
                want = plain / 4 * ramp + plain * (1 - ramp)
        assert abs(f - want) <= 1e-12 * want + 1e-15, i
    assert t.scale == pytest.approx(0.1 * math.log(4.0) + 1.0 if name == "yarn" else 1.0)


def test_operators_refuse_host_tensors():
    from glq_b200 import ops
    x = torch.zeros(2, 4, 64, dtype=torch.bfloat16)
    c = torch.zeros(3, 16, 2, 64, dtype=torch.bfloat16)
    n = torch.zeros(2, dtype=torch.int64)
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        ops.rotary(x, n, None)
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        ops.paged_append(x[:, :2], x[:, :2], c, c, n)
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        ops.paged_attention(x, c, c, torch.zeros(2, 1, dtype=torch.int32), n)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.rotary_table(64, device="cpu")
    for bad in (dict(dim=7), dict(dim=0), dict(), dict(dim=8, scaling={"rope_type": "other", "factor": 2.0}), dict(dim=8, scaling={"rope_type": "linear"}),
                dict(dim=8, scaling={"rope_type": "yarn", "factor": 2.0}), dict(dim=8, inv_freq=torch.ones(3)), dict(inv_freq=torch.tensor([math.inf]))):
        with pytest.raises(ValueError, match="glq_b200"):
            ops.rotary_table(**bad)


def test_operators_refuse_wrong_arguments(monkeypatch):
    """The checks behind the one for the device, on host tensors; nothing is launched."""
    from glq_b200 import ops, paged
    table = _table(monkeypatch, 32)
    big = _table(monkeypatch, 128)
    monkeypatch.setattr(paged, "_cuda", lambda t, name: None)
    monkeypatch.setattr(paged, "_same_device", lambda t, x, name: None)
    monkeypatch.setattr(paged, "_device_of", lambda t, name, index=None: -1)
    launched = []
    monkeypatch.setattr(paged, "_call", lambda *a: launched.append(a[1]))
    monkeypatch.setattr(paged, "_workspace", lambda *a: 64)
    bf = torch.bfloat16
    x, n3 = torch.zeros(3, 4, 64, dtype=bf), torch.zeros(3, dtype=torch.int64)

    def refuses(text, fn, *a, **kw):
        with pytest.raises(ValueError, match=text):
            fn(*a, **kw)

    refuses("tokens, heads", ops.rotary, x[0], n3, table)
    refuses("not torch.float64", ops.rotary, x.double(), n3, table)
    refuses("rotary_table", ops.rotary, x, n3, None)
    refuses("128 rotated values", ops.rotary, x, n3, big)
    refuses("positions must be 3", ops.rotary, x, n3[:2], table)
    refuses("positions must be 3", ops.rotary, x, n3.float(), table)
    refuses("out must be", ops.rotary, x, n3, table, out=x[:2])
    refuses("overlap", ops.rotary, x, n3, table, out=x[:1].expand(3, 4, 64))
    refuses("without being it", ops.rotary, x, n3, table, out=torch.as_strided(x, x.shape, (64, 192, 1)))
    y = torch.zeros(3, 64, 4, dtype=bf).transpose(1, 2)
    refuses("one behind the other", ops.rotary, y, n3, table, out=y)

    k, v = (torch.zeros(5, 16, 2, 64, dtype=bf) for _ in range(2))
    new = torch.zeros(3, 2, 64, dtype=bf)
    refuses("one type", ops.paged_append, new, new, k, v.half(), n3)
    refuses("one type", ops.paged_append, new, new, k, v[:4], n3)
    refuses("bf16 or fp16", ops.paged_append, new, new, k.float(), v.float(), n3)
    refuses("power of two", ops.paged_append, new, new, k[:, :12], v[:, :12], n3)
    refuses("multiple of 8", ops.paged_append, new[..., :12], new[..., :12], k[..., :12], v[..., :12], n3)
    refuses("16 bytes", ops.paged_append, new, new, k.transpose(1, 3).contiguous().transpose(1, 3), v, n3)
    refuses("for a cache of", ops.paged_append, new[:, :1], new[:, :1], k, v, n3)
    refuses("for a cache of", ops.paged_append, new, new[:2], k, v, n3)
    refuses("fp32", ops.paged_append, new.half(), new.half(), k, v, n3)
    refuses("slots must be 3", ops.paged_append, new, new, k, v, n3[:1])
    refuses("come together", ops.paged_append, new, new, k, v, n3, table=table)
    refuses("come together", ops.paged_append, new, new, k, v, n3, positions=n3)
    refuses("to be rotated", ops.paged_append, new, new, k, v, n3, query=x)
    refuses("belongs to query", ops.paged_append, new, new, k, v, n3, out=x)
    refuses("beside keys", ops.paged_append, new, new, k, v, n3, positions=n3, table=table, query=x.float())
    refuses("beside keys", ops.paged_append, new, new, k, v, n3, positions=n3, table=table, query=x[:2])
    refuses("128 rotated", ops.paged_append, new, new, k, v, n3, positions=n3, table=big)
    refuses("out overlaps key", ops.paged_append, new, torch.zeros_like(new), k, v, n3, positions=n3, table=table, query=torch.zeros_like(new), out=new)
    refuses("overlaps the cache", ops.paged_append, new, k[0, :3], k, v, n3)
    # parts of a merged projection lie between each other's rows: they may be rotated in place, but not onto one another
    merged = torch.zeros(3, 8, 64, dtype=bf)
    q, kk, vv = merged[:, :4], merged[:, 4:6], merged[:, 6:]
    assert ops.paged_append(kk, vv, k, v, n3, positions=n3, table=table, query=q, out=q) is q and launched.pop() == "paged_append"
    assert ops.rotary(merged[:, :2], n3, table, out=merged[:, 5:7]) is not None and launched.pop() == "rotary"
    refuses("out overlaps key", ops.paged_append, merged[:, 3:5], vv, k, v, n3, positions=n3, table=table, query=q, out=q)
    refuses("out overlaps key", ops.paged_append, kk, merged[:, 1:3], k, v, n3, positions=n3, table=table, query=q, out=q)
    refuses("without being it", ops.rotary, merged[:, :2], n3, table, out=merged[:, 1:3])

    pages = torch.zeros(3, 2, dtype=torch.int32)
    ok = (x, k, v, pages, n3)
    refuses("over a cache", ops.paged_attention, x.half(), *ok[1:])
    refuses("over a cache", ops.paged_attention, x[:, :3], *ok[1:])
    refuses("over a cache", ops.paged_attention, x[..., :32], *ok[1:])
    refuses("pages must be int32", ops.paged_attention, x, k, v, pages.long(), n3)
    refuses("pages must be int32", ops.paged_attention, x, k, v, pages.t().contiguous().t(), n3)
    refuses("lengths must be 3", ops.paged_attention, x, k, v, pages, n3[:2])
    refuses("query_offsets must be 4", ops.paged_attention, *ok, query_offsets=n3)
    refuses("need query_offsets", ops.paged_attention, x, k, v, pages[:2], n3[:2])
    refuses("max_query_len", ops.paged_attention, *ok, max_query_len=-1)
    for scale in (0.0, -0.5, math.nan, math.inf):
        refuses("positive", ops.paged_attention, *ok, scale=scale)
    for window in (-1, 2 ** 31):
        refuses("window", ops.paged_attention, *ok, window=window)
    refuses("out must be", ops.paged_attention, *ok, out=x.half())
    refuses("overlaps", ops.paged_attention, *ok, out=x)
    assert not launched
    ops.rotary(x, n3, table)
    ops.paged_append(new, new, k, v, n3, positions=n3, table=table, query=x)
    ops.paged_attention(*ok)
    assert launched == ["rotary", "paged_append", "paged_attention"]
    # expanded queries go to the device as copies, which every kernel can read
    packed = []
    real = paged._lib.pack_attention
    monkeypatch.setattr(paged._lib, "pack_attention", lambda *a: packed.append(a[2:4]) or real(*a))
    ops.paged_attention(x[:, :1].expand(3, 4, 64), *ok[1:])
    ops.paged_attention(x[:1].expand(3, 4, 64), *ok[1:])
    assert packed == [(256, 64)] * 2


def _model(lengths, new, group, kv_heads, rows, keys, ctas, begin, least, causal=True, window=0):
    """How attention's work is shared out: a list of units, `begin` for an item and one per key tile of it, cut into equal runs, of `least`
    units if there are as many.  The items as (sequence, key head, row tile, lo, hi) and what the CTAs have of them as (cta, item, lo, hi, slot, begun_by, parts)."""
    items = []
    for s, (n, q) in enumerate(zip(lengths, new)):
        for h in range(kv_heads):
            for t in range(-(-q * group // rows)):
                last = min(q - 1, (min(q * group, (t + 1) * rows) - 1) // group)
                first = t * rows // group
                to = max(0, n - q + last + 1) if causal else n
                lo = min(to, max(0, n - q + first + 1 - window) if window else 0) // keys
                items.append((s, h, t, lo, max(lo + 1, -(-to // keys))))
    total = sum(i[4] - i[3] + begin for i in items)
    used = min(ctas, -(-total // least))
    cta_of = lambda u: ((u + 1) * used - 1) // total
    out, at = [], 0
    for i, (s, h, t, lo, hi) in enumerate(items):
        for c in range(cta_of(at), cta_of(at + begin + hi - lo - 1) + 1):
            x = max(0, total * c // used - at - begin)
            y = min(hi - lo, total * (c + 1) // used - at - begin)
            if x < y:
                slot = -1 if y - x == hi - lo else 0 if x else 1
                first = at + begin
                out.append((c, i, lo + x, lo + y, slot, cta_of(first), cta_of(first + hi - lo - 1) - cta_of(first) + 1))
        at += begin + hi - lo
    return items, out


@pytest.mark.parametrize("lengths,new", [([4096], [1]), ([100, 3, 900, 0, 64], [1] * 5), ([700, 2], [650, 2]), ([5000], [5000]), ([31, 64, 1] * 50, [1] * 150)])
@pytest.mark.parametrize("rows,keys,ctas,begin,least", [(16, 64, 296, 2, 3), (256, 128, 148, 2, 4), (16, 64, 7, 2, 3), (256, 128, 5, 0, 1)])
@pytest.mark.parametrize("window", [0, 200])
def test_runs_cover_the_work_and_parts_find_their_item(lengths, new, rows, keys, ctas, begin, least, window):
    """Every key tile is taken once.  Of an item that is cut, the CTA that all take for its first leaves its part in slot 1 and the others, the CTAs behind
    it without a gap, theirs in slot 0; all know how many they are."""
    items, runs = _model(lengths, new, 4, 2, rows, keys, ctas, begin, least, window=window)
    slots, cut = set(), set()
    for c, i, lo, hi, slot, begun_by, parts in runs:
        if slot >= 0:
            assert (c, slot) not in slots                        # a CTA leaves at most one part in either slot
            slots.add((c, slot))
    for i, (s, h, t, lo, hi) in enumerate(items):
        mine = [r for r in runs if r[1] == i]
        assert mine[0][2] == lo and mine[-1][3] == hi and all(a[3] == b[2] for a, b in zip(mine, mine[1:]))
        if len(mine) == 1:
            assert mine[0][4] == -1
            continue
        assert [r[4] for r in mine] == [1] + [0] * (len(mine) - 1)
        assert [r[0] for r in mine] == list(range(mine[0][0], mine[0][0] + len(mine)))
        assert all(r[5] == mine[0][0] and r[6] == len(mine) for r in mine)
        assert mine[0][0] not in cut                             # (a ticket is that CTA's: one item that it begins and does not end)
        cut.add(mine[0][0])


@pytest.fixture(scope="module")
def the_list(tmp_path_factory):
    """The kernels' own list of work, built for the host."""
    from glq_b200 import build
    out = str(tmp_path_factory.mktemp("list") / "list.so")
    res = subprocess.run([build._nvcc(), *build.NVCC_FLAGS, "-O1", "-I", build.CSRC, "-I", os.path.join(ROOT, "include"), os.path.join(ROOT, "tests", "paged_list.cu"), "-o", out],
                         capture_output=True, text=True)
    assert res.returncode == 0, res.stderr
    fn = ctypes.CDLL(out).paged_list

    def rows(lengths, new, group, kv_heads, rows, keys, grid, begin, least, causal=True, window=0):
        offsets = [sum(new[:i]) for i in range(len(new) + 1)]
        numbers, most = (ctypes.c_int * (14 << 16))(), 1 << 16
        n = fn((ctypes.c_longlong * len(lengths))(*lengths), (ctypes.c_longlong * len(offsets))(*offsets), len(lengths), offsets[-1], 1 << 30, group, kv_heads, rows, keys, grid, begin,
               least, int(causal), window, numbers, most)
        assert 0 <= n < most
        return [tuple(numbers[14 * i:14 * i + 14]) for i in range(n)]

    return rows


@pytest.mark.parametrize("lengths,new", [([4096], [1]), ([100, 3, 900, 0, 64], [1] * 5), ([700, 2], [650, 2]), ([5000], [5000]), ([31, 64, 1] * 50, [1] * 150),
                                         ([0, 5, 130, 400, 64, 1, 700, 129], [0, 5, 1, 33, 64, 1, 2, 0]), ([3, 0, 70], [10, 4, 200]), ([9], [0])])
@pytest.mark.parametrize("rows,keys,ctas,begin,least", [(16, 64, 296, 2, 3), (240, 128, 148, 2, 4), (256, 128, 148, 2, 4), (16, 64, 7, 2, 3), (256, 128, 5, 0, 1)])
@pytest.mark.parametrize("causal,window", [(True, 0), (True, 200), (False, 0), (False, 30)])
def test_kernels_share_work_as_the_model_does(the_list, lengths, new, rows, keys, ctas, begin, least, causal, window):
    """Item for item, and that no query of an item sees a key outside its tiles."""
    group = 5 if rows == 240 else 4
    items, runs = _model(lengths, new, group, 2, rows, keys, ctas, begin, least, causal, window) if sum(new) else ([], [])
    got = the_list(lengths, new, group, 2, rows, keys, ctas, begin, least, causal, window)
    assert len(got) == len(runs)
    covered = {}
    for (c, i, lo, hi, slot, begun_by, parts), row in zip(sorted(runs), got):
        s, h, t, first_tile, last_tile = items[i]
        assert row[:3] == (c, s, h) and row[3] == t * rows and row[4] == min(rows, new[s] * group - t * rows) and row[5:8] == (lo, hi, slot)
        assert slot < 0 or row[8:10] == (begun_by, parts)
        # keys of the item's first and last query
        ends = []
        for q in (row[3] // group, (row[3] + row[4] - 1) // group):
            at = lengths[s] - new[s] + q
            ends.append((max(0, at + 1 - window) if window else 0, max(0, at + 1) if causal else lengths[s]))
        (f0, t0), (f1, t1) = ends
        assert row[10:] == (f1, t0, f0, t1)
        assert t1 <= f0 or first_tile * keys <= f0 and t1 <= last_tile * keys
        covered.setdefault(i, []).append((lo, hi))
    assert len(covered) == len(items)
